// dash_norm.cu -- the residual sum behind a block, with the block's own norm, its
// gate and scale, and the norm before the next block; forward and gradients.
//
//   z = y * r1 * post            r1 = 1 / sqrt(mean(y^2) + eps)   (post given; else z = y)
//   s = residual + scale * gate * z
//   h = s * r2 * weight          r2 = 1 / sqrt(mean(s^2) + eps)
//
// All arithmetic is fp32; s and h are rounded once each (h is made of the unrounded
// s).  The gradients make s again from y and the residual, so that nothing but the
// inputs is kept, and no rounded s enters the weights' gradients.
//
// Bound by memory: y and residual in, s and h out (forward); those two and the
// gradients of s and h in, those of y and residual out (backward).  Rows of 1,280, bf16: forward
// 36,992 of them 66 us (5.8 TB/s; 78 with post and gate), 8 of them 5.2 us from a graph;
// gradients of 9,248 plain ones 27 us (22 at the copy rate), of 36,992 with post and gate 143 us
// (87, the column sums' kernel among them).  With post or gate the forward's issue of instructions is 72% busy and memory 52%;
// in the gradients the issue of instructions is 60% busy with 15 warps on an SM, which is what the
// column sums and weights in registers leave room for.
#include "dash_common.cuh"
#include "dash_internal.h"

namespace dash {

namespace {

constexpr int kNormMaxHidden = 8192;

// E consecutive elements as fp32
template <typename T, int E>
struct Row;
template <typename T>
struct Row<T, 1> {
  T v;
  __device__ __forceinline__ void read(const T* p) { v = *p; }
  __device__ __forceinline__ void get(float (&x)[1]) const { x[0] = (float)v; }
  __device__ __forceinline__ void put(const float (&x)[1]) { v = (T)x[0]; }
  __device__ __forceinline__ void write(T* p) const { *p = v; }
};
template <typename T>
struct Row<T, 8> {            // 16-bit types
  uint4 v;
  __device__ __forceinline__ void read(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(w[i], (T*)nullptr);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  __device__ __forceinline__ void put(const float (&x)[8]) {
    v = make_uint4(pack2(x[0], x[1], (T*)nullptr), pack2(x[2], x[3], (T*)nullptr), pack2(x[4], x[5], (T*)nullptr),
                   pack2(x[6], x[7], (T*)nullptr));
  }
  __device__ __forceinline__ void write(T* p) const { *reinterpret_cast<uint4*>(p) = v; }
};
template <>
struct Row<float, 4> {
  float4 v;
  __device__ __forceinline__ void read(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w; }
  __device__ __forceinline__ void put(const float (&x)[4]) { v = make_float4(x[0], x[1], x[2], x[3]); }
  __device__ __forceinline__ void write(float* p) const { *reinterpret_cast<float4*>(p) = v; }
};

// E elements of a weight that is fp32 or of the rows' type
template <typename T, int E>
__device__ __forceinline__ void read_weight(const void* p, int64_t at, bool f32, float (&x)[E]) {
  if (f32) {
    const float* w = static_cast<const float*>(p) + at;
    if constexpr (E == 1) {
      x[0] = *w;
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(w + i);
        x[i] = f.x, x[i + 1] = f.y, x[i + 2] = f.z, x[i + 3] = f.w;
      }
    }
  } else {
    Row<T, E> r;
    r.read(static_cast<const T*>(p) + at);
    r.get(x);
  }
}

// Sums of N values over a row's threads, the same in all of them: a warp's by
// shuffles, then the warps' in their order.  `buf` alternates between two halves, so
// that one barrier per call is enough.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int warps, int warp, int lane, float* buf, int& half) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if (warps == 1) return;
  float* b = buf + half * 32 * 5;
  half ^= 1;
  if (lane == 0)
#pragma unroll
    for (int n = 0; n < N; ++n) b[n * 32 + warp] = v[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float s = 0.0f;
    for (int w = 0; w < warps; ++w) s += b[n * 32 + w];
    v[n] = s;
  }
}

template <typename T, int E, int NV>
__global__ void __launch_bounds__(512) add_norm_kernel(const DashNormArgs a, int warps) {
  __shared__ float buf[2 * 32 * 5];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // one warp per row, several rows per CTA; or the whole CTA on one row
  const int64_t row = warps == 1 ? (int64_t)blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x;
  if (row >= a.rows) return;
  const int t = warps == 1 ? lane : (int)threadIdx.x, step = warps * 32 * E;
  int half = 0;
  const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
  const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
  Row<T, E> ry[NV], rr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t * E + i * step;
    if (c < a.hidden) ry[i].read(y + c);
    if (res && c < a.hidden) rr[i].read(res + c);
  }
  const float inv = 1.0f / (float)a.hidden;
  float r1 = 1.0f;
  if (a.post) {
    float q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t * E + i * step < a.hidden) {
        float x[E];
        ry[i].get(x);
#pragma unroll
        for (int e = 0; e < E; ++e) q[0] = fmaf(x[e], x[e], q[0]);
      }
    row_sum(q, warps, warp, lane, buf, half);
    r1 = rsqrtf(q[0] * inv + a.eps);
  }
  const int64_t group = a.gate ? row / a.group_rows : 0;
  float s[NV][E], q[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t * E + i * step;
    if (c < a.hidden) {
      ry[i].get(s[i]);
      if (a.post) {
        float p[E];
        read_weight<T, E>(a.post, c, a.post_f32, p);
#pragma unroll
        for (int e = 0; e < E; ++e) s[i][e] *= r1 * p[e];
      }
      if (a.gate) {
        float g[E];
        read_weight<T, E>(a.gate, group * a.gate_stride + c, a.gate_f32, g);
#pragma unroll
        for (int e = 0; e < E; ++e) s[i][e] *= g[e];
      }
      float r[E] = {};
      if (res) rr[i].get(r);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s[i][e] = fmaf(s[i][e], a.scale, r[e]);
        q[0] = fmaf(s[i][e], s[i][e], q[0]);
      }
    }
  }
  row_sum(q, warps, warp, lane, buf, half);
  const float r2 = rsqrtf(q[0] * inv + a.eps);
  T* so = a.stream ? static_cast<T*>(a.stream) + row * a.stream_stride : nullptr;
  T* ho = static_cast<T*>(a.normed) + row * a.normed_stride;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t * E + i * step;
    if (c < a.hidden) {
      Row<T, E> o;
      if (so) {
        o.put(s[i]);
        o.write(so + c);
      }
      float w[E];
      read_weight<T, E>(a.weight, c, a.weight_f32, w);
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] *= s[i][e] * r2;
      o.put(w);
      o.write(ho + c);
    }
  }
}

// Gradients.  With a = dh * weight and sh = s * r2,
//   ds_total = ds + r2 * (a - sh * mean(a * sh))         (the residual's gradient)
//   dweight  = sum over rows of dh * sh
//   dz       = scale * gate * ds_total,  dgate = sum over the group's rows of scale * z * ds_total
//   dy       = dz;  with post, b = dz * post and yh = y * r1:  dy = r1 * (b - yh * mean(b * yh)),
//              dpost = sum over rows of dz * yh
// mean(b * yh) = r1 / n * sum(q * ds_total) with q = scale * gate * post * y, which splits into the
// sums of q * ds, q * a and q * s: one exchange between the warps per row (two with post).
//
// A CTA takes whole rows, a thread the same columns of each, so the column sums stay in
// registers; rows go to CTAs in chunks that lie within one gate's group.  Column sums of
// a CTA (dweight, dpost) and of a chunk (dgate) are written to the workspace and added
// in their order by norm_columns_kernel: no atomics.  This form is for rows that are not
// aligned to 16 bytes, and for the longest fp32 rows.
template <typename T, int E, int NV>
__global__ void __launch_bounds__(512) add_norm_bwd_kernel(const DashNormBwdArgs b, int64_t chunk, int64_t chunks_per_group, int64_t chunks,
                                    float* part_w, float* part_p, float* part_g) {
  const DashNormArgs& a = b.fwd;
  __shared__ float buf[2 * 32 * 5];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int t = threadIdx.x, step = (int)blockDim.x * E;
  int half = 0;
  const float inv = 1.0f / (float)a.hidden;
  float dw[NV][E] = {}, dp[NV][E] = {};
  for (int64_t k = blockIdx.x; k < chunks; k += gridDim.x) {
    const int64_t group = k / chunks_per_group, piece = k % chunks_per_group;
    const int64_t end = min((group + 1) * a.group_rows, group * a.group_rows + (piece + 1) * chunk);
    float dg[NV][E] = {};
    for (int64_t row = group * a.group_rows + piece * chunk; row < end; ++row) {
      const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
      const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
      const T* gs = b.dstream ? static_cast<const T*>(b.dstream) + row * b.dstream_stride : nullptr;
      const T* gh = static_cast<const T*>(b.dnormed) + row * b.dnormed_stride;
      Row<T, E> ry[NV], rr[NV], rs[NV], rh[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t * E + i * step;
        if (c < a.hidden) {
          ry[i].read(y + c);
          if (res) rr[i].read(res + c);
          if (gs) rs[i].read(gs + c);
          rh[i].read(gh + c);
        }
      }
      float r1 = 1.0f;
      if (a.post) {
        float q[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (t * E + i * step < a.hidden) {
            float x[E];
            ry[i].get(x);
#pragma unroll
            for (int e = 0; e < E; ++e) q[0] = fmaf(x[e], x[e], q[0]);
          }
        row_sum(q, warps, warp, lane, buf, half);
        r1 = rsqrtf(q[0] * inv + a.eps);
      }
      // f = scale * gate, q = f * post * y: s = residual + q * r1
      float f[NV][E], p[NV][E], s[NV][E], ga[NV][E];
      float sum[5] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t * E + i * step;
        if (c < a.hidden) {
          float x[E], r[E] = {}, d[E] = {};
#pragma unroll
          for (int e = 0; e < E; ++e) f[i][e] = 1.0f, p[i][e] = 1.0f;
          if (a.gate) read_weight<T, E>(a.gate, group * a.gate_stride + c, a.gate_f32, f[i]);
          if (a.post) read_weight<T, E>(a.post, c, a.post_f32, p[i]);
          read_weight<T, E>(a.weight, c, a.weight_f32, ga[i]);
          ry[i].get(x);
          if (res) rr[i].get(r);
          rh[i].get(s[i]);
          if (gs) rs[i].get(d);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            f[i][e] *= a.scale;
            ga[i][e] *= s[i][e];
            const float q = f[i][e] * p[i][e] * x[e];
            s[i][e] = fmaf(q, r1, r[e]);
            sum[0] = fmaf(s[i][e], s[i][e], sum[0]);
            sum[1] = fmaf(ga[i][e], s[i][e], sum[1]);
            sum[2] = fmaf(q, d[e], sum[2]);
            sum[3] = fmaf(q, ga[i][e], sum[3]);
            sum[4] = fmaf(q, s[i][e], sum[4]);
          }
        }
      }
      if (a.post) {
        row_sum(sum, warps, warp, lane, buf, half);
      } else {
        float two[2] = {sum[0], sum[1]};
        row_sum(two, warps, warp, lane, buf, half);
        sum[0] = two[0], sum[1] = two[1];
      }
      const float r2 = rsqrtf(sum[0] * inv + a.eps);
      // ds_total = ds + r2 * a - m * s, dy = r1 * (b - mb * yh)   (multiplied in turn: r1 and r2 to the
      // third power leave the range of fp32 where the rows are around 2^43 or 2^-43)
      const float m = r2 * (r2 * (r2 * sum[1]) * inv);
      const float mb = r1 * (sum[2] + r2 * sum[3] - m * sum[4]) * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t * E + i * step;
        if (c < a.hidden) {
          float x[E], d[E] = {}, hh[E], o[E];
          ry[i].get(x);
          if (gs) rs[i].get(d);
          rh[i].get(hh);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            d[e] = fmaf(r2, ga[i][e], d[e]) - m * s[i][e];
            dw[i][e] = fmaf(hh[e], s[i][e] * r2, dw[i][e]);
            const float dz = d[e] * f[i][e], yh = x[e] * r1;
            dg[i][e] = fmaf(d[e], a.scale * yh * p[i][e], dg[i][e]);
            dp[i][e] = fmaf(dz, yh, dp[i][e]);
            o[e] = a.post ? r1 * fmaf(-mb, yh, dz * p[i][e]) : dz;
          }
          Row<T, E> w;
          if (b.dresidual) {
            w.put(d);
            w.write(static_cast<T*>(b.dresidual) + row * b.dresidual_stride + c);
          }
          if (b.dy) {
            w.put(o);
            w.write(static_cast<T*>(b.dy) + row * b.dy_stride + c);
          }
        }
      }
    }
    if (part_g) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t * E + i * step;
        if (c < a.hidden)
#pragma unroll
          for (int e = 0; e < E; ++e) part_g[k * a.hidden + c + e] = dg[i][e];
      }
    } else if (b.dgate) {                       // the chunk is a whole group
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t * E + i * step;
        if (c < a.hidden)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            if (a.gate_f32) static_cast<float*>(b.dgate)[k * a.hidden + c + e] = dg[i][e];
            else static_cast<T*>(b.dgate)[k * a.hidden + c + e] = (T)dg[i][e];
          }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t * E + i * step;
    if (c < a.hidden)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        part_w[(int64_t)blockIdx.x * a.hidden + c + e] = dw[i][e];
        if (part_p) part_p[(int64_t)blockIdx.x * a.hidden + c + e] = dp[i][e];
      }
  }
}

// The same for aligned rows.  What bounded the form above at 36,992 rows of 1,280 (bf16, gate and
// post: 234 us, memory takes 87) were instructions and the two exchanges per row, not
// the loads, so here
//  - two elements share an instruction (f32x2),
//  - a row's exchange carries the sum of squares that the next row's r1 is made of,
//  - sums are folded together before they are shuffled (9 shuffles for 6 sums, not 30),
//  - the next rows are on their way into shared memory (cp.async; a thread fetches what it
//    reads itself, so they need no barrier).
template <int NV>
constexpr int kAhead = NV == 1 ? 3 : 1;            // rows on their way: 128 KB of shared memory at most
constexpr int kRingMost = 128 * 1024;
constexpr int kRingPlain = 46 * 1024;              // without asking for more: 48 KB with the static part

__device__ __forceinline__ uint64_t fmul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t both(float x) { return f2_pack(x, x); }
__device__ __forceinline__ float add_up(uint64_t v) {
  float x, y;
  f2_unpack(v, x, y);
  return x + y;
}

// 16 bytes as pairs of fp32, and back
template <typename T>
struct Pairs {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint64_t get(const uint4& v, int j) {
    const uint32_t w = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
    const float2 f = unpack2(w, (T*)nullptr);
    return f2_pack(f.x, f.y);
  }
  static __device__ __forceinline__ void put(uint4& v, int j, uint64_t x) {
    float a, b;
    f2_unpack(x, a, b);
    const uint32_t w = pack2(a, b, (T*)nullptr);
    (j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w) = w;
  }
};
template <>
struct Pairs<float> {
  static constexpr int N = 2;
  static __device__ __forceinline__ uint64_t get(const uint4& v, int j) {
    return j ? f2_pack(__uint_as_float(v.z), __uint_as_float(v.w)) : f2_pack(__uint_as_float(v.x), __uint_as_float(v.y));
  }
  static __device__ __forceinline__ void put(uint4& v, int j, uint64_t x) {
    float a, b;
    f2_unpack(x, a, b);
    (j ? v.z : v.x) = __float_as_uint(a);
    (j ? v.w : v.y) = __float_as_uint(b);
  }
};

// Sums of N (2 or 8) values over a row's threads, the same in all of them.  At each step
// the lanes send the half of the values that they will not keep.
template <int N>
__device__ __forceinline__ void fold(float (&v)[N], int warps, int warp, int lane, float* buf, int& half) {
  float x = 0.0f;
  int mine;
  if constexpr (N == 2) {
    const bool up = lane & 16;
    x = (up ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, up ? v[0] : v[1], 16);
    mine = 16;
  } else {
    float f[4], g[2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = (lane & 16 ? v[4 + i] : v[i]) + __shfl_xor_sync(0xffffffffu, lane & 16 ? v[i] : v[4 + i], 16);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      g[i] = (lane & 8 ? f[2 + i] : f[i]) + __shfl_xor_sync(0xffffffffu, lane & 8 ? f[i] : f[2 + i], 8);
    x = (lane & 4 ? g[1] : g[0]) + __shfl_xor_sync(0xffffffffu, lane & 4 ? g[0] : g[1], 4);
    mine = 4;
  }
  for (int o = mine / 2; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  float* b = buf + half * 16 * 8;
  half ^= 1;
  if ((lane & (mine - 1)) == 0) b[warp * 8 + lane / mine] = x;
  if (warps > 1) __syncthreads();
  else __syncwarp();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.0f;
  for (int w = 0; w < warps; ++w) {
    if constexpr (N == 2) {
      const float2 s = *reinterpret_cast<const float2*>(b + w * 8);
      v[0] += s.x, v[1] += s.y;
    } else {
      const float4 s = *reinterpret_cast<const float4*>(b + w * 8), t = *reinterpret_cast<const float4*>(b + w * 8 + 4);
      v[0] += s.x, v[1] += s.y, v[2] += s.z, v[3] += s.w;
      v[4] += t.x, v[5] += t.y, v[6] += t.z, v[7] += t.w;
    }
  }
}

// FULL: with post, gate or both
template <typename T, int NV, bool FULL>
__global__ void __launch_bounds__(512) add_norm_bwd_wide_kernel(const DashNormBwdArgs b, int64_t chunk, int64_t chunks_per_group,
                                                                int64_t chunks, float* part_w, float* part_p, float* part_g) {
  constexpr int E = 16 / sizeof(T), P = Pairs<T>::N, AHEAD = kAhead<NV>, F = FULL ? NV : 1;
  const DashNormArgs& a = b.fwd;
  __shared__ __align__(16) float buf[2 * 16 * 8];
  extern __shared__ uint4 ring[];                // [AHEAD + 1][4][NV][threads]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int t = threadIdx.x, step = (int)blockDim.x * E, plane = NV * (int)blockDim.x;
  const bool post = FULL && a.post, gate = FULL && a.gate;
  int half = 0;
  const float inv = 1.0f / (float)a.hidden;
  uint64_t dw[NV][P] = {}, dp[F][P] = {}, dg[F][P], w[NV][P], p[F][P], g[F][P];
  const auto pairs_of = [&](const void* from, int64_t at, bool f32, uint64_t (&to)[P]) {
    float x[E];
    read_weight<T, E>(from, at, f32, x);
#pragma unroll
    for (int j = 0; j < P; ++j) to[j] = f2_pack(x[2 * j], x[2 * j + 1]);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t * E + i * step;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      w[i][j] = 0;
      if (FULL) p[FULL ? i : 0][j] = both(1.0f);
    }
    if (c < a.hidden) {
      pairs_of(a.weight, c, a.weight_f32, w[i]);
      if (post) pairs_of(a.post, c, a.post_f32, p[FULL ? i : 0]);
    }
  }
  // the row to be fetched next, in this CTA's order
  int64_t fk = blockIdx.x, frow = 0, fend = 0;
  const auto open = [&](int64_t k, int64_t& row, int64_t& end) {
    const int64_t group = k / chunks_per_group;
    row = group * a.group_rows + (k - group * chunks_per_group) * chunk;
    end = min((group + 1) * a.group_rows, row + chunk);
  };
  const auto fetch = [&](int slot) {
    if (fk < chunks) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t * E + i * step;
        const uint32_t to = smem_u32(ring + (slot * 4 * NV + i) * (int)blockDim.x + t);
        const auto copy = [&](int n, const void* from, int64_t stride) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + n * plane * 16),
                       "l"(static_cast<const T*>(from) + frow * stride + c)
                       : "memory");
        };
        if (c < a.hidden) {
          copy(0, a.y, a.y_stride);
          if (a.residual) copy(1, a.residual, a.residual_stride);
          if (b.dstream) copy(2, b.dstream, b.dstream_stride);
          copy(3, b.dnormed, b.dnormed_stride);
        }
      }
      if (++frow == fend && (fk += gridDim.x) < chunks) open(fk, frow, fend);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  open(fk, frow, fend);
  for (int n = 0; n < AHEAD; ++n) fetch(n);
  // what lies behind the row's end, or has no tensor, counts as 0
  const auto read = [&](int slot, int n, int i, bool on) {
    return on && t * E + i * step < a.hidden ? ring[(slot * 4 + n) * plane + i * (int)blockDim.x + t] : make_uint4(0, 0, 0, 0);
  };
  const auto squares = [&](int slot) {           // of this thread's part of y
    uint64_t q = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint4 v = read(slot, 0, i, true);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const uint64_t x = Pairs<T>::get(v, j);
        q = ffma2(x, x, q);
      }
    }
    return add_up(q);
  };
  int at = 0;                                    // the ring's row in use
  float next = 0.0f;                             // sum of squares of the row that comes next
  bool known = false;
  for (int64_t k = blockIdx.x; k < chunks; k += gridDim.x) {
    int64_t row, end;
    open(k, row, end);
    if (FULL) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        constexpr int I = FULL ? 1 : 0;
        const int c = t * E + i * step;
#pragma unroll
        for (int j = 0; j < P; ++j) g[I * i][j] = both(1.0f), dg[I * i][j] = 0;
        if (gate && c < a.hidden) pairs_of(a.gate, k / chunks_per_group * a.gate_stride + c, a.gate_f32, g[I * i]);
#pragma unroll
        for (int j = 0; j < P; ++j) g[I * i][j] = fmul2(g[I * i][j], both(a.scale));
      }
    }
    for (; row < end; ++row) {
      // this row is there, and with three rows on their way the next one too
      asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD >= 3 ? AHEAD - 2 : AHEAD - 1) : "memory");
      const int after = at == AHEAD ? 0 : at + 1;
      if (post && !(AHEAD >= 3 && known)) {
        float q[2] = {squares(at), 0.0f};
        fold(q, warps, warp, lane, buf, half);
        next = q[0];
        known = true;
      }
      const float r1 = post ? rsqrtf(next * inv + a.eps) : 1.0f;
      uint4 ry[NV], rs[NV], rh[NV];
      uint64_t s[NV][P], sum[5] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        constexpr int I = FULL ? 1 : 0;
        ry[i] = read(at, 0, i, true);
        rs[i] = read(at, 2, i, b.dstream);
        rh[i] = read(at, 3, i, true);
        const uint4 rr = read(at, 1, i, a.residual);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const uint64_t ga = fmul2(w[i][j], Pairs<T>::get(rh[i], j));
          const uint64_t q = fmul2(FULL ? fmul2(g[I * i][j], p[I * i][j]) : both(a.scale), Pairs<T>::get(ry[i], j));
          s[i][j] = ffma2(q, both(r1), Pairs<T>::get(rr, j));
          sum[0] = ffma2(s[i][j], s[i][j], sum[0]);
          sum[1] = ffma2(ga, s[i][j], sum[1]);
          if (FULL) {
            sum[2] = ffma2(q, Pairs<T>::get(rs[i], j), sum[2]);
            sum[3] = ffma2(q, ga, sum[3]);
            sum[4] = ffma2(q, s[i][j], sum[4]);
          }
        }
      }
      float v[8] = {add_up(sum[0]), add_up(sum[1])};
      if (post) {
        v[2] = add_up(sum[2]), v[3] = add_up(sum[3]), v[4] = add_up(sum[4]);
        if (AHEAD >= 3) v[5] = squares(after);
        fold(v, warps, warp, lane, buf, half);
        next = v[5];
      } else {
        float two[2] = {v[0], v[1]};
        fold(two, warps, warp, lane, buf, half);
        v[0] = two[0], v[1] = two[1];
      }
      // (the slot that is filled now was read before the exchange)
      fetch(at == 0 ? AHEAD : at - 1);
      at = after;
      const float r2 = rsqrtf(v[0] * inv + a.eps);
      const float m = r2 * (r2 * (r2 * v[1]) * inv);            // ds_total = ds + r2 * ga - m * s (in turn, as above)
      const float mb = r1 * (v[2] + r2 * v[3] - m * v[4]) * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        constexpr int I = FULL ? 1 : 0;
        const int c = t * E + i * step;
        uint4 od, oy;
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const uint64_t h = fmul2(Pairs<T>::get(rh[i], j), both(r2));
          uint64_t d = ffma2(w[i][j], h, Pairs<T>::get(rs[i], j));
          d = ffma2(both(-m), s[i][j], d);
          dw[i][j] = ffma2(h, s[i][j], dw[i][j]);
          Pairs<T>::put(od, j, d);
          if (FULL) {
            const uint64_t x = Pairs<T>::get(ry[i], j), yh = fmul2(x, both(r1)), dz = fmul2(d, g[I * i][j]);
            dg[I * i][j] = ffma2(d, fmul2(yh, p[I * i][j]), dg[I * i][j]);
            dp[I * i][j] = ffma2(dz, yh, dp[I * i][j]);
            Pairs<T>::put(oy, j, post ? fmul2(ffma2(yh, both(-mb), fmul2(dz, p[I * i][j])), both(r1)) : dz);
          } else {
            Pairs<T>::put(oy, j, fmul2(d, both(a.scale)));
          }
        }
        if (c < a.hidden) {
          if (b.dresidual) *reinterpret_cast<uint4*>(static_cast<T*>(b.dresidual) + row * b.dresidual_stride + c) = od;
          if (b.dy) *reinterpret_cast<uint4*>(static_cast<T*>(b.dy) + row * b.dy_stride + c) = oy;
        }
      }
    }
    if (FULL && b.dgate) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t * E + i * step;
        if (c < a.hidden)
#pragma unroll
          for (int j = 0; j < P; ++j) {
            float x[2];
            f2_unpack(fmul2(dg[FULL ? i : 0][j], both(a.scale)), x[0], x[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int64_t o = k * a.hidden + c + 2 * j + e;
              if (part_g) part_g[o] = x[e];
              else if (a.gate_f32) static_cast<float*>(b.dgate)[o] = x[e];     // the chunk is a whole group
              else static_cast<T*>(b.dgate)[o] = (T)x[e];
            }
          }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t * E + i * step;
    if (c < a.hidden)
#pragma unroll
      for (int j = 0; j < P; ++j) {
        *reinterpret_cast<uint64_t*>(part_w + (int64_t)blockIdx.x * a.hidden + c + 2 * j) = dw[i][j];
        if (FULL && part_p) *reinterpret_cast<uint64_t*>(part_p + (int64_t)blockIdx.x * a.hidden + c + 2 * j) = dp[FULL ? i : 0][j];
      }
  }
}

// The forward with post or gate in the same manner, for many aligned rows: a CTA takes rows one after the other,
// its weights stay in registers.
template <typename T, int NV>
__global__ void __launch_bounds__(512) add_norm_wide_kernel(const DashNormArgs a, int64_t per) {
  constexpr int E = 16 / sizeof(T), P = Pairs<T>::N, AHEAD = kAhead<NV>;
  __shared__ __align__(16) float buf[2 * 16 * 8];
  extern __shared__ uint4 ring[];                // [AHEAD + 1][2][NV][threads]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int t = threadIdx.x, step = (int)blockDim.x * E, plane = NV * (int)blockDim.x;
  const bool post = a.post, gate = a.gate;
  const int64_t first = blockIdx.x * per, end = min(a.rows, first + per);
  int half = 0;
  const float inv = 1.0f / (float)a.hidden;
  uint64_t w[NV][P], p[NV][P], g[NV][P];
  const auto pairs_of = [&](const void* from, int64_t at, bool f32, uint64_t (&to)[P]) {
    float x[E];
    read_weight<T, E>(from, at, f32, x);
#pragma unroll
    for (int j = 0; j < P; ++j) to[j] = f2_pack(x[2 * j], x[2 * j + 1]);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t * E + i * step;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      w[i][j] = 0;
      p[i][j] = both(1.0f);
    }
    if (c < a.hidden) {
      pairs_of(a.weight, c, a.weight_f32, w[i]);
      if (post) pairs_of(a.post, c, a.post_f32, p[i]);
    }
  }
  int64_t frow = first;
  const auto fetch = [&](int slot) {
    if (frow < end) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t * E + i * step;
        const uint32_t to = smem_u32(ring + (slot * 2 * NV + i) * (int)blockDim.x + t);
        const auto copy = [&](int n, const void* from, int64_t stride) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + n * plane * 16),
                       "l"(static_cast<const T*>(from) + frow * stride + c)
                       : "memory");
        };
        if (c < a.hidden) {
          copy(0, a.y, a.y_stride);
          if (a.residual) copy(1, a.residual, a.residual_stride);
        }
      }
      ++frow;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int n = 0; n < AHEAD; ++n) fetch(n);
  const auto read = [&](int slot, int n, int i, bool on) {
    return on && t * E + i * step < a.hidden ? ring[(slot * 2 + n) * plane + i * (int)blockDim.x + t] : make_uint4(0, 0, 0, 0);
  };
  const auto squares = [&](int slot) {
    uint64_t q = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint4 v = read(slot, 0, i, true);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const uint64_t x = Pairs<T>::get(v, j);
        q = ffma2(x, x, q);
      }
    }
    return add_up(q);
  };
  int at = 0;
  float next = 0.0f;
  bool known = false;
  int64_t border = first;                        // the row at which another gate begins
  for (int64_t row = first; row < end; ++row) {
    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD >= 3 ? AHEAD - 2 : AHEAD - 1) : "memory");
    const int after = at == AHEAD ? 0 : at + 1;
    if (row == border) {
      const int64_t group = row / a.group_rows;
      border = (group + 1) * a.group_rows;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t * E + i * step;
#pragma unroll
        for (int j = 0; j < P; ++j) g[i][j] = both(1.0f);
        if (gate && c < a.hidden) pairs_of(a.gate, group * a.gate_stride + c, a.gate_f32, g[i]);
#pragma unroll
        for (int j = 0; j < P; ++j) g[i][j] = fmul2(fmul2(g[i][j], p[i][j]), both(a.scale));
      }
    }
    if (post && !(AHEAD >= 3 && known)) {
      float q[2] = {squares(at), 0.0f};
      fold(q, warps, warp, lane, buf, half);
      next = q[0];
      known = true;
    }
    const uint64_t r1 = both(post ? rsqrtf(next * inv + a.eps) : 1.0f);
    uint64_t s[NV][P], sum = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint4 y = read(at, 0, i, true), r = read(at, 1, i, a.residual);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const uint64_t q = fmul2(g[i][j], Pairs<T>::get(y, j));
        s[i][j] = ffma2(q, r1, Pairs<T>::get(r, j));
        sum = ffma2(s[i][j], s[i][j], sum);
      }
    }
    float v[2] = {add_up(sum), post && AHEAD >= 3 ? squares(after) : 0.0f};
    fold(v, warps, warp, lane, buf, half);
    next = v[1];
    fetch(at == 0 ? AHEAD : at - 1);
    at = after;
    const uint64_t r2 = both(rsqrtf(v[0] * inv + a.eps));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t * E + i * step;
      uint4 os, oh;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        Pairs<T>::put(os, j, s[i][j]);
        Pairs<T>::put(oh, j, fmul2(fmul2(s[i][j], r2), w[i][j]));
      }
      if (c < a.hidden) {
        if (a.stream) *reinterpret_cast<uint4*>(static_cast<T*>(a.stream) + row * a.stream_stride + c) = os;
        *reinterpret_cast<uint4*>(static_cast<T*>(a.normed) + row * a.normed_stride + c) = oh;
      }
    }
  }
}

// out[g][c] = sum over j of part[g * n + j][c], in that order: 32 columns per CTA, the
// parts dealt to its warps
template <typename T>
__device__ __forceinline__ void columns(const float* part, int64_t n, int hidden, int64_t g, void* out, bool f32) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (c < hidden)
    for (int64_t j = warp; j < n; j += 32) v += part[(g * n + j) * hidden + c];
  s[warp][lane] = v;
  __syncthreads();
  v = s[lane][warp];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int oc = blockIdx.x * 32 + warp;
  if (lane == 0 && oc < hidden) {
    if (f32) static_cast<float*>(out)[g * hidden + oc] = v;
    else static_cast<T*>(out)[g * hidden + oc] = (T)v;
  }
}

// blockIdx.y: 0 dweight, 1 dpost, then the gate's groups
template <typename T>
__global__ void __launch_bounds__(1024) norm_columns_kernel(const DashNormBwdArgs b, const float* part_w,
                                                           const float* part_p, const float* part_g, int ctas,
                                                           int64_t chunks_per_group) {
  const DashNormArgs& a = b.fwd;
  const int64_t first = part_p ? 2 : 1;
  if (blockIdx.y == 0) {
    if (b.dweight) columns<T>(part_w, ctas, a.hidden, 0, b.dweight, a.weight_f32);
  } else if (blockIdx.y < first) {
    if (b.dpost) columns<T>(part_p, ctas, a.hidden, 0, b.dpost, a.post_f32);
  } else {
    for (int64_t g = blockIdx.y - first; g < a.rows / a.group_rows; g += gridDim.y - first) {
      columns<T>(part_g, chunks_per_group, a.hidden, g, b.dgate, a.gate_f32);
      __syncthreads();
    }
  }
}

template <typename T, int E>
bool wide(const DashNormArgs& a) {
  const auto ok = [](const void* p, int64_t stride, int64_t unit) {
    return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % unit == 0);
  };
  return a.hidden % E == 0 && ok(a.y, a.y_stride, E) && ok(a.residual, a.residual_stride, E) &&
         ok(a.stream, a.stream_stride, E) && ok(a.normed, a.normed_stride, E) && ok(a.weight, 0, 1) &&
         ok(a.post, 0, 1) && ok(a.gate, a.gate_stride, E);
}

// The forward with post or gate takes a CTA per row where each CTA has a few of them: 36,992
// rows of 1,280 (bf16) 78 us, a warp per row 89.  Without them a warp per row takes 66
// us, a CTA 68.
constexpr int kFwdRows = 4, kFwdThreads = 1536;

template <typename T, int E>
int launch_fwd_e(const DashNormArgs& a, cudaStream_t st) {
  const int vecs = (a.hidden + E - 1) / E;
  if constexpr (E > 1) {
    const int nv = vecs <= 512 ? 1 : 2, threads = (vecs + 32 * nv - 1) / (32 * nv) * 32;
    const int64_t ctas = 148 * max(1, min(12, kFwdThreads / threads));
    if ((a.post || a.gate) && threads <= 512 && threads >= 64 && a.rows >= kFwdRows * ctas) {
      const int64_t per = (a.rows + ctas - 1) / ctas;
      const unsigned grid = (unsigned)((a.rows + per - 1) / per);
      const size_t ring = (size_t)(nv == 1 ? kAhead<1> + 1 : kAhead<2> + 1) * 2 * nv * threads * 16;
      const auto go = [&](auto kernel) {
        if (ring > kRingPlain && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingMost) != cudaSuccess)
          return set_error(DASH_ERR_CUDA, "add_norm_kernel: no shared memory for the ring");
        kernel<<<grid, threads, ring, st>>>(a, per);
        count_launch();
        return check_launch("add_norm_kernel");
      };
      return nv == 1 ? go(add_norm_wide_kernel<T, 1>) : go(add_norm_wide_kernel<T, 2>);
    }
  }
  // A warp holds a row of up to 8 vectors per lane (no barrier); longer rows get the
  // whole CTA.
  const int warps = vecs <= 256 ? 1 : min(16, (vecs + 127) / 128);
  const int nv = (vecs + warps * 32 - 1) / (warps * 32);
  const int threads = warps == 1 ? 128 : warps * 32;
  const unsigned grid = (unsigned)(warps == 1 ? (a.rows + 3) / 4 : a.rows);
  if (nv <= 2) add_norm_kernel<T, E, 2><<<grid, threads, 0, st>>>(a, warps);
  else if (nv <= 4) add_norm_kernel<T, E, 4><<<grid, threads, 0, st>>>(a, warps);
  else if (nv <= 8) add_norm_kernel<T, E, 8><<<grid, threads, 0, st>>>(a, warps);
  else if constexpr (E == 1) add_norm_kernel<T, E, 16><<<grid, threads, 0, st>>>(a, warps);
  count_launch();
  return check_launch("add_norm_kernel");
}

constexpr int kNormThreads = 512;                  // of a backward call on an SM: 128 registers each

// How the rows of a backward call are dealt out
struct NormCut {
  int threads, nv, ctas;
  int64_t chunk, per_group, chunks;
};

NormCut norm_cut(const DashNormArgs& a, int E) {
  NormCut c;
  const int vecs = (a.hidden + E - 1) / E;
  // One vector per thread up to 256 of them; more vectors per thread, then 512
  // threads, for longer rows (the column sums live in registers).
  c.nv = 1;
  int warps = (vecs + 31) / 32;
  for (const int most : {8, 16})
    while (warps > most && c.nv < (E == 1 ? (most == 8 ? 8 : 16) : most == 8 ? 8 / E : 16 / E))
      c.nv *= 2, warps = (vecs + 32 * c.nv - 1) / (32 * c.nv);
  c.threads = warps * 32;
  const int most = 148 * max(1, min(8, kNormThreads / c.threads));
  // rows dealt evenly, in chunks that lie within a group
  const int64_t groups = a.rows / a.group_rows;
  const int64_t want = (a.rows + most - 1) / most;
  c.chunk = min((int64_t)a.group_rows, max((int64_t)1, want));
  c.per_group = (a.group_rows + c.chunk - 1) / c.chunk;
  c.chunks = groups * c.per_group;
  c.ctas = (int)min((int64_t)most, c.chunks);
  return c;
}

template <typename T, int E>
int launch_bwd_e(const DashNormBwdArgs& b, cudaStream_t st) {
  const DashNormArgs& a = b.fwd;
  const NormCut c = norm_cut(a, E);
  float* part_w = static_cast<float*>(b.workspace);
  float* part_p = a.post ? part_w + (int64_t)c.ctas * a.hidden : nullptr;
  float* part_g = b.dgate && c.per_group > 1 ? part_w + (int64_t)c.ctas * a.hidden * (a.post ? 2 : 1) : nullptr;
  const auto go = [&](auto kernel, size_t ring) {
    if (ring > kRingPlain && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingMost) != cudaSuccess)
      return set_error(DASH_ERR_CUDA, "add_norm_bwd_kernel: no shared memory for the ring");
    kernel<<<c.ctas, c.threads, ring, st>>>(b, c.chunk, c.per_group, c.chunks, part_w, part_p, part_g);
    return (int)DASH_OK;
  };
  const size_t row = (size_t)4 * c.nv * c.threads * 16;
  const bool full = a.post || a.gate;
  int rr = DASH_OK;
  if constexpr (E == 1) {
    rr = c.nv == 1   ? go(add_norm_bwd_kernel<T, E, 1>, 0)
         : c.nv == 2 ? go(add_norm_bwd_kernel<T, E, 2>, 0)
         : c.nv == 4 ? go(add_norm_bwd_kernel<T, E, 4>, 0)
         : c.nv == 8 ? go(add_norm_bwd_kernel<T, E, 8>, 0)
                     : go(add_norm_bwd_kernel<T, E, 16>, 0);
  } else if (c.nv == 1) {
    const size_t ring = row * (kAhead<1> + 1);
    rr = full ? go(add_norm_bwd_wide_kernel<T, 1, true>, ring) : go(add_norm_bwd_wide_kernel<T, 1, false>, ring);
  } else if (c.nv == 2) {
    const size_t ring = row * (kAhead<2> + 1);
    rr = full ? go(add_norm_bwd_wide_kernel<T, 2, true>, ring) : go(add_norm_bwd_wide_kernel<T, 2, false>, ring);
  } else if constexpr (E == 4) {
    rr = go(add_norm_bwd_kernel<T, E, 4>, 0);
  }
  if (rr) return rr;
  count_launch();
  int rc = check_launch("add_norm_bwd_kernel");
  if (rc) return rc;
  const int64_t groups = part_g ? a.rows / a.group_rows : 0;
  const dim3 grid((a.hidden + 31) / 32, (unsigned)((a.post ? 2 : 1) + min(groups, (int64_t)4096)));
  norm_columns_kernel<T><<<grid, 1024, 0, st>>>(b, part_w, part_p, part_g, c.ctas, c.per_group);
  count_launch();
  return check_launch("norm_columns_kernel");
}

bool norm_bwd_wide(const DashNormBwdArgs& b, int E) {
  const auto ok = [E](const void* p, int64_t stride) {
    return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % E == 0);
  };
  return ok(b.dstream, b.dstream_stride) && ok(b.dnormed, b.dnormed_stride) && ok(b.dy, b.dy_stride) &&
         ok(b.dresidual, b.dresidual_stride);
}

}  // namespace

int launch_add_norm(const DashNormArgs& a, cudaStream_t st) {
  if (a.dtype == DASH_DTYPE_F32) return wide<float, 4>(a) ? launch_fwd_e<float, 4>(a, st) : launch_fwd_e<float, 1>(a, st);
  if (a.dtype == DASH_DTYPE_BF16)
    return wide<__nv_bfloat16, 8>(a) ? launch_fwd_e<__nv_bfloat16, 8>(a, st) : launch_fwd_e<__nv_bfloat16, 1>(a, st);
  return wide<__half, 8>(a) ? launch_fwd_e<__half, 8>(a, st) : launch_fwd_e<__half, 1>(a, st);
}

static bool bwd_is_wide(const DashNormBwdArgs& b) {
  if (b.fwd.dtype == DASH_DTYPE_F32) return wide<float, 4>(b.fwd) && norm_bwd_wide(b, 4);
  return wide<__half, 8>(b.fwd) && norm_bwd_wide(b, 8);
}

size_t add_norm_bwd_workspace(const DashNormBwdArgs& b) {
  const DashNormArgs& a = b.fwd;
  // whichever vector width the pointers allow
  size_t most = 0;
  for (const int E : {1, a.dtype == DASH_DTYPE_F32 ? 4 : 8}) {
    const NormCut c = norm_cut(a, E);
    const size_t n = (size_t)a.hidden * ((size_t)c.ctas * (a.post ? 2 : 1) + (a.gate && c.per_group > 1 ? (size_t)c.chunks : 0));
    if (n > most) most = n;
  }
  return most * sizeof(float);
}

int launch_add_norm_bwd(const DashNormBwdArgs& b, cudaStream_t st) {
  const bool w = bwd_is_wide(b);
  if (b.fwd.dtype == DASH_DTYPE_F32) return w ? launch_bwd_e<float, 4>(b, st) : launch_bwd_e<float, 1>(b, st);
  if (b.fwd.dtype == DASH_DTYPE_BF16)
    return w ? launch_bwd_e<__nv_bfloat16, 8>(b, st) : launch_bwd_e<__nv_bfloat16, 1>(b, st);
  return w ? launch_bwd_e<__half, 8>(b, st) : launch_bwd_e<__half, 1>(b, st);
}

int norm_max_hidden() { return kNormMaxHidden; }

}  // namespace dash
