// dash_tree.cuh -- one (drafted token, query head) of the draft-tree attention
// by one warp on the CUDA cores: the rows of block sizes that the tensor-core
// kernel does not tile, and the rows that it hands back because a value that
// is not finite reached their sums (dash_tree_tc.cu).
//
// A warp is 4 groups of 8 lanes; group g takes keys g, g + 4, ... of a range,
// lane `sub` 16 of the 128 dims.  Every group keeps a running maximum and sum;
// the groups are merged at the end.  Logits and maximum are in natural units,
// where every bias of the type has its place: times log2(e) the lowest ones
// would be -inf.  Only keys that the row attends are read, so what lies in
// other rows of a page cannot reach it.
#pragma once
#include "dash_common.cuh"
#include "dash_internal.h"

namespace dash {

constexpr float kTreeLog2e = 1.4426950408889634f;
constexpr float kTreeLn2 = 0.6931471805599453f;

struct TreeSeq {
  int64_t row0;   // first packed row
  int n;          // drafted tokens
  int ctx;        // committed tokens
};

// Drafted tokens of sequence s, cut to the rows and the count that the call allows.
__device__ __forceinline__ TreeSeq tree_seq(const int32_t* q_start, const int32_t* ctx_len, int rows, int max_nodes,
                                            int s) {
  TreeSeq t;
  const int a = q_start[s];
  t.row0 = a;
  t.n = a < 0 ? 0 : max(0, min(min(q_start[s + 1], rows) - a, max_nodes));
  t.ctx = min(max(0, ctx_len[s]), INT32_MAX / 2);
  return t;
}

// The sequence of packed row r (r < q_start[n_seq]); empty sequences own no row.
__device__ __forceinline__ int tree_seq_of_row(const int32_t* q_start, int n_seq, int64_t r) {
  int lo = 0, hi = n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (q_start[mid] <= r) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void tree_unpack8(const uint4 w, float* x, __nv_bfloat16* t) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = unpack2(ws[e], t);
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
}
__device__ __forceinline__ void tree_unpack8(const uint4 w, float* x, __half* t) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = unpack2(ws[e], t);
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
}

// A lane's 16 dims of a query row, from its first dim's 16-byte piece and the next.
template <typename T>
__device__ __forceinline__ void tree_load_q(const uint4& lo, const uint4& hi, float (&q)[16]) {
  tree_unpack8(lo, q, (T*)nullptr);
  tree_unpack8(hi, q + 8, (T*)nullptr);
}

// Attention of packed row r (token of sequence s) and query head hq, whose dims
// [16 sub, 16 sub + 16) the caller has read into q; the whole warp calls it.  On
// return every lane holds the row's maximum m (-inf without a key), sum l and its
// dims of the unscaled output, the same in all four groups.
template <typename T>
__device__ void tree_row_attend(const DashTreeAttnArgs& a, const TreeSeq& sq, int s, int64_t r, int hq,
                                float (&q)[16], float scale, float& m, float& l, float (&o)[16]) {
  const int lane = threadIdx.x & 31, grp = lane >> 3, sub = lane & 7;
  const int H = a.qo.n_heads, hk = hq / (H / a.kv.n_kv_heads), bs = a.block_size;
  const int nih = a.routes.n_index_heads > 0 ? a.routes.n_index_heads : 1;
  const int64_t roff = r * a.routes.row_stride + (int64_t)(hq / (H / nih)) * a.routes.ihead_stride;
  const T* kp = reinterpret_cast<const T*>(a.kv.k) + (int64_t)hk * a.kv.stride_head + sub * 16;
  const T* vp = reinterpret_cast<const T*>(a.kv.v) + (int64_t)hk * a.kv.stride_head + sub * 16;
  const int32_t* bt = a.kv.block_table + (int64_t)s * a.kv.bt_stride;
#pragma unroll
  for (int c = 0; c < 16; ++c) q[c] *= scale;
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int c = 0; c < 16; ++c) o[c] = 0.0f;

  auto page_of = [&](int b) -> int64_t {
    const int64_t p = b < a.bt_width ? (int64_t)bt[b] : -1;
    if (p >= 0 && p < a.kv.num_pages) return p;
    if (lane == 0) record_error(a.device_error, DASH_DEV_BAD_PAGE, 70, p);
    return -1;
  };
  // keys [t0, t1) of block b with the bias b2; vis != null: only
  // the drafted tokens whose bit is set there (token u is key sq.ctx + u)
  auto block = [&](int b, int t0, int t1, float b2, const uint32_t* vis) {
    if (t1 <= t0) return;
    const int64_t p = page_of(b);
    if (p < 0) return;
    const int64_t base = p * a.kv.stride_seq - (int64_t)b * bs * a.kv.stride_tok;
    for (int t = t0; t < t1; t += 4) {
      const int j = t + grp;
      bool on = j < t1;
      if (on && vis) {
        const int u = j - sq.ctx;
        on = (u >> 5) < a.mask_words && ((vis[u >> 5] >> (u & 31)) & 1u);
      }
      float sc = 0.0f, v[16];
      if (on) {
        float k[16];
        const int64_t off = base + (int64_t)j * a.kv.stride_tok;
        const uint4* k4 = reinterpret_cast<const uint4*>(kp + off);
        const uint4* v4 = reinterpret_cast<const uint4*>(vp + off);
        tree_unpack8(__ldg(k4), k, (T*)nullptr);
        tree_unpack8(__ldg(k4 + 1), k + 8, (T*)nullptr);
        tree_unpack8(__ldg(v4), v, (T*)nullptr);
        tree_unpack8(__ldg(v4 + 1), v + 8, (T*)nullptr);
#pragma unroll
        for (int c = 0; c < 16; ++c) sc = fmaf(q[c], k[c], sc);
      }
      sc += __shfl_xor_sync(0xffffffffu, sc, 1);
      sc += __shfl_xor_sync(0xffffffffu, sc, 2);
      sc += __shfl_xor_sync(0xffffffffu, sc, 4);
      if (on) {
        sc += b2;
        const float mn = fmaxf(m, sc);
        if (mn != -INFINITY || sc != sc) {
          const float al = m == -INFINITY ? 0.0f : fast_exp2((m - mn) * kTreeLog2e);
          const float p = fast_exp2((sc - mn) * kTreeLog2e);
          l = l * al + p;
#pragma unroll
          for (int c = 0; c < 16; ++c) o[c] = fmaf(p, v[c], o[c] * al);
          m = mn;
        }
      }
    }
  };

  const int64_t edge = (int64_t)a.row_pos[r] - a.local_window + 1;          // first key of the window
  const int lstart = (int)max((int64_t)0, min(edge, (int64_t)sq.ctx));
  const int nblk = (sq.ctx + sq.n + bs - 1) / bs;
  for (int j = 0; j < a.routes.K; ++j) {
    const int b = a.routes.idx[roff + j];
    if (b < 0) continue;
    if (b >= nblk) {
      if (lane == 0) record_error(a.device_error, DASH_DEV_BAD_BLOCK, 71, b);
      continue;
    }
    bool again = false;                                                      // the first occurrence counts
    for (int u = lane; u < j; u += 32) again |= a.routes.idx[roff + u] == b;
    if (__any_sync(0xffffffffu, again)) continue;
    const float b2 = a.routes.bias ? a.routes.bias[roff + j] : 0.0f;
    if (b2 == -INFINITY) continue;                                           // masked: nothing in it counts
    const int t0 = (int)min((int64_t)b * bs, (int64_t)lstart);
    block(b, t0, (int)min((int64_t)(b + 1) * bs, (int64_t)lstart), b2, nullptr);
  }
  for (int t = lstart; t < sq.ctx;) {
    const int b = t / bs, t1 = (int)min((int64_t)(b + 1) * bs, (int64_t)sq.ctx);
    block(b, t, t1, 0.0f, nullptr);
    t = t1;
  }
  const uint32_t* vis = a.mask + r * a.mask_stride;
  for (int t = sq.ctx; t < sq.ctx + sq.n;) {
    const int b = t / bs, t1 = (int)min((int64_t)(b + 1) * bs, (int64_t)sq.ctx + sq.n);
    block(b, t, t1, 0.0f, vis);
    t = t1;
  }
  // join the groups (lanes of equal sub); NaN stays in l and o, the maximum skips it
#pragma unroll
  for (int off = 8; off < 32; off <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, off), l2 = __shfl_xor_sync(0xffffffffu, l, off);
    const float mn = fmaxf(m, m2);
    const float fa = m == -INFINITY ? (l == l ? 0.0f : 1.0f) : fast_exp2((m - mn) * kTreeLog2e);
    const float fb = m2 == -INFINITY ? (l2 == l2 ? 0.0f : 1.0f) : fast_exp2((m2 - mn) * kTreeLog2e);
    l = l * fa + l2 * fb;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const float o2 = __shfl_xor_sync(0xffffffffu, o[c], off);
      o[c] = o[c] * fa + o2 * fb;
    }
    m = mn;
  }
}

// The lanes of group 0 store the row's output and its natural-log sum.
template <typename T>
__device__ __forceinline__ void tree_row_store(const DashTreeAttnArgs& a, int64_t r, int hq, float m, float l,
                                               const float (&o)[16]) {
  const int lane = threadIdx.x & 31;
  if (lane >= 8) return;
  const bool none = l == 0.0f;                      // no key: 0, -inf (a NaN sum is not "none")
  const float inv = none ? 0.0f : 1.0f / l;
  T* op = reinterpret_cast<T*>(a.qo.out) + r * a.qo.o_stride_tok + (int64_t)hq * a.qo.o_stride_head + lane * 16;
  uint32_t w[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) w[c] = pack2(none ? 0.0f : o[2 * c] * inv, none ? 0.0f : o[2 * c + 1] * inv, (T*)nullptr);
  *reinterpret_cast<uint4*>(op) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(op + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  if (lane == 0 && a.qo.lse)
    a.qo.lse[r * a.qo.lse_stride_tok + (int64_t)hq * a.qo.lse_stride_head] =
        none ? -INFINITY : m + log2f(l) * kTreeLn2;
}

}  // namespace dash
