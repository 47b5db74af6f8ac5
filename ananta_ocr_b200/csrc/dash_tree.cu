// dash_tree.cu -- draft trees on the paged cache: the plan (positions, masks,
// cache slots from the parents) and the attention's CUDA-core form (one warp
// per drafted token and query head, dash_tree.cuh).
#include "dash_tree.cuh"

namespace dash {

constexpr int kTreeMaxNodes = 256;

// One CTA per sequence, one thread per drafted token: a token's parents are
// before it, so its chain of ancestors ends after at most `depth` reads of the
// shared parent list.  Latency-bound (a few hundred bytes per sequence).
__global__ void __launch_bounds__(kTreeMaxNodes) tree_plan_kernel(const DashTreePlanArgs a) {
  __shared__ int s_par[kTreeMaxNodes];
  const int s = blockIdx.x, i = threadIdx.x;
  const TreeSeq sq = tree_seq(a.q_start, a.ctx_len, a.rows, a.max_nodes, s);
  if (i == 0 && a.q_start[s + 1] - a.q_start[s] > a.max_nodes)
    record_error(a.device_error, DASH_DEV_BAD_TREE, 72, a.q_start[s + 1] - a.q_start[s]);
  const int64_t r = sq.row0 + i;
  if (i < sq.n) {
    int p = a.parents ? a.parents[r] : i - 1;
    if (i == 0) p = -1;
    if (p < 0 || p >= i) {
      if (i > 0) record_error(a.device_error, DASH_DEV_BAD_TREE, 73, p);
      p = -1;
    }
    s_par[i] = p;
  }
  __syncthreads();
  if (i >= sq.n) return;
  uint32_t m[kTreeMaxNodes / 32];
#pragma unroll
  for (int w = 0; w < kTreeMaxNodes / 32; ++w) m[w] = (i >> 5) == w ? 1u << (i & 31) : 0u;
  int depth = 0;
  for (int p = s_par[i]; p >= 0; p = s_par[p]) {
    ++depth;
#pragma unroll
    for (int w = 0; w < kTreeMaxNodes / 32; ++w) m[w] |= (p >> 5) == w ? 1u << (p & 31) : 0u;
  }
  if (a.depth) a.depth[r] = depth;
  if (a.row_pos) a.row_pos[r] = sq.ctx + depth;
  if (a.row_seq) a.row_seq[r] = s;
  if (a.mask)
#pragma unroll
    for (int w = 0; w < kTreeMaxNodes / 32; ++w)
      if (w < a.mask_words) a.mask[r * a.mask_words + w] = m[w];
  if (a.slots) {
    const int t = sq.ctx + i, b = t / a.block_size;
    int64_t page = b < a.bt_width ? (int64_t)a.block_table[(int64_t)s * a.bt_stride + b] : -1;
    if (page < 0 || page >= a.num_pages) {
      record_error(a.device_error, DASH_DEV_BAD_PAGE, 74, page);
      page = -1;
    }
    a.slots[r] = page < 0 ? -1 : page * a.block_size + t % a.block_size;
  }
}

int launch_tree_plan(const DashTreePlanArgs& a, cudaStream_t st) {
  tree_plan_kernel<<<a.n_seq, kTreeMaxNodes, 0, st>>>(a);
  count_launch();
  return check_launch("tree_plan_kernel");
}

constexpr int kTreeRowWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kTreeRowWarps * 32) tree_rows_kernel(const __grid_constant__ DashTreeAttnArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * kTreeRowWarps + (threadIdx.x >> 5);
  const int64_t r = unit / a.qo.n_heads;
  const int hq = (int)(unit - r * a.qo.n_heads);
  if (r >= a.seqs.q_len_fixed || r >= a.seqs.q_start[a.seqs.n_seq] || r < a.seqs.q_start[0]) return;
  const int s = tree_seq_of_row(a.seqs.q_start, a.seqs.n_seq, r);
  const TreeSeq sq = tree_seq(a.seqs.q_start, a.ctx_len, a.seqs.q_len_fixed, a.seqs.max_q_len, s);
  if (r - sq.row0 >= sq.n) return;
  const uint4* qp = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.qo.q) + r * a.qo.q_stride_tok +
                                                   (int64_t)hq * a.qo.q_stride_head + (threadIdx.x & 7) * 16);
  float q[16], m, l, o[16];
  tree_load_q<T>(qp[0], qp[1], q);
  tree_row_attend<T>(a, sq, s, r, hq, q, a.scale, m, l, o);
  tree_row_store<T>(a, r, hq, m, l, o);
}

// The tensor cores wherever the block size lets a 64-key tile be made of granules: the
// CUDA-core form reads every key once per row and head, and took five times as long or
// more: 474 us where the other takes 78 (32 sequences of one token on 27,556), 280 / 47 (16 trees of 16), 100 / 20.5
// (8 of 17), 83 / 14.5 (one of 8), 618 / 33 (four of 64).
int launch_tree_attn(const DashTreeAttnArgs& a, cudaStream_t st) {
  if (tree_tc_supported(a)) return launch_tree_tc(a, st);
  const int64_t units = (int64_t)a.seqs.q_len_fixed * a.qo.n_heads;
  const unsigned grid = (unsigned)((units + kTreeRowWarps - 1) / kTreeRowWarps);
  if (a.kv.dtype == DASH_DTYPE_BF16)
    tree_rows_kernel<__nv_bfloat16><<<grid, kTreeRowWarps * 32, 0, st>>>(a);
  else
    tree_rows_kernel<__half><<<grid, kTreeRowWarps * 32, 0, st>>>(a);
  count_launch();
  return check_launch("tree_rows_kernel");
}

}  // namespace dash
