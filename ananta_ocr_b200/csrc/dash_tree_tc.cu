// dash_tree_tc.cu -- draft-tree attention on the sm_100a tensor cores.
//
// Work unit: up to 128 (drafted token, query head) rows of one sequence and kv
// head, split over a cluster of 1..8 CTAs.  The keys that any row attends --
// the union of the rows' routed blocks, their windows and the drafted tokens --
// are cut into granules of GR tokens (GR = block size, 64 at most); a tile of 64
// keys is 64 / GR granules of the union in ascending order, and each CTA of the
// cluster takes a contiguous part of the tiles.  Every key of the union crosses
// the memory bus once per kv head, whatever the number of drafted tokens, which is
// what bounds the kernel: 32 KB of K and V per tile against ~0.5 k cycles of
// tensor work (M = 128 rows, padded) and ~0.6 k of softmax per SM sub-partition.
//
//   setup (all)       union bit set and its prefix sums in shared memory
//   warp 4  TMA       block table -> page boxes {64 dims, GR tokens} of K and V
//                     (128-byte swizzle), K and V in rings of their own (2 x
//                     16 KB each): a K slot is free after Q K^T, a V slot after P V
//   warp 5  MMA       S = Q K^T (M 128, N 64, two TMEM buffers), O += P V (N 128, P
//                     from TMEM)
//   warps 0-3 softmax one thread per row; warps without a row sleep.  The additive
//                     terms of the routed granules lie in a [granule][token]
//                     table (first occurrence of a repeated id by atomicMin on
//                     the slot), refilled when a part outgrows it
//
// 96 KB of Q, K and V stages and 256 TMEM columns per CTA: two CTAs per SM, whose
// phases interleave.  At the end the CTAs leave O, the running maximum and the
// sum in their shared memory and each joins its share of the rows over the
// cluster (no workspace, no atomics, fixed order).
//
// A masked key has P = 0, and 0 * v is 0 only for finite v.  V rows behind the last
// drafted token are zeroed; a row whose joined output is not finite for any
// other reason (a bad value in a key that some other row attends, or in its own)
// is computed again from its own keys only (tree_row_attend), so no row
// depends on keys that it does not attend.
#include <cooperative_groups.h>
#include <cudaTypedefs.h>
#include "dash_tree.cuh"

namespace cg = cooperative_groups;

namespace dash {
namespace {

constexpr int kRows = 128;                       // M of both MMAs
constexpr int kKeys = 64;                        // N of Q K^T, K of P V
constexpr int kThreads = 192;
constexpr int kStages = 2;
constexpr int kSlot = 16384;                     // one tile of K or of V: 2 x [64 x 128 B]
constexpr int kCells = 3000;                     // additive terms held at a time
constexpr int kMaxWords = 512;                   // 16384 granules of a sequence
constexpr uint32_t kTmemCols = 256;              // S0 | S1 | O
constexpr float kGrow = 8.0f;                    // O is rescaled when a row's maximum grows by 2^8

struct TreeSmem {
  uint8_t q[2 * kRows * 128];                    // two halves of 64 dims, swizzled
  uint8_t k[kStages][kSlot];                     // k and v together receive O (128 x 512 B) at the end
  uint8_t v[kStages][kSlot];
  float cell[kCells];
  uint32_t bits[kMaxWords];
  uint16_t before[kMaxWords + 1];
  int tok[kStages][4];                           // first token of the tile's granules, -1 = none
  float m[kRows], l[kRows];
  uint64_t kfull[kStages], kempty[kStages], vfull[kStages], vempty[kStages];
  uint64_t sfull[2], pfull[2], pvdone[2], qfull, alldone;
  uint32_t tmem;
  int abort_flag;
};
static_assert(offsetof(TreeSmem, v) == offsetof(TreeSmem, k) + kStages * kSlot, "O spans the K and V slots");
static_assert(kStages * kSlot * 2 == kRows * 512, "O spans the K and V slots");
static_assert(sizeof(TreeSmem) + 1024 <= 233472 / 2 - 1024, "two CTAs per SM");

// the j-th set bit of w (j < popc(w))
__device__ __forceinline__ int nth_bit(uint32_t w, int j) { return (int)__fns(w, 0, j + 1); }

}  // namespace

template <typename T, int GR>
__global__ void __launch_bounds__(kThreads, 2)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ DashTreeAttnArgs a, int n_tiles_seq) {
  constexpr int NG = kKeys / GR;                 // granules per tile
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  TreeSmem& S = *reinterpret_cast<TreeSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  cg::cluster_group cluster = cg::this_cluster();
  const int nsp = (int)cluster.num_blocks(), split = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int u = blockIdx.x / nsp;
  const int tile_i = u % n_tiles_seq;
  u /= n_tiles_seq;
  const int hk = u % a.kv.n_kv_heads, s = u / a.kv.n_kv_heads;
  const int H = a.qo.n_heads, G = H / a.kv.n_kv_heads, bs = a.block_size;
  const int per_tile = kRows / G;                // tokens of a tile
  TreeSeq sq = tree_seq(a.seqs.q_start, a.ctx_len, a.seqs.q_len_fixed, a.seqs.max_q_len, s);
  const int node0 = tile_i * per_tile;
  const int nt = min(per_tile, sq.n - node0);    // this tile's tokens
  if (nt <= 0) return;                           // the whole cluster leaves
  const int total_n = sq.n;
  const int64_t r0 = sq.row0 + node0;            // packed row of the tile's first token
  const int nrows = nt * G, nact = (nrows + 31) >> 5;
  const int nih = a.routes.n_index_heads > 0 ? a.routes.n_index_heads : 1;
  const int64_t ioff = (int64_t)((hk * G) / (H / nih)) * a.routes.ihead_stride;
  const int K = a.routes.K;
  DeviceError* derr = a.device_error;
  const int ctx = sq.ctx, end = ctx + total_n;
  // tokens behind the table's last column do not exist
  const int64_t room = (int64_t)a.bt_width * bs;
  const int words = min(kMaxWords, (int)((min((int64_t)end, room) + 32 * GR - 1) / (32 * GR)));
  if ((int64_t)end > room && tid == 0 && hk == 0 && split == 0) record_error(derr, DASH_DEV_BAD_PAGE, 75, a.bt_width);
  const int live_end = (int)min((int64_t)end, room);
  const int nblk = (end + bs - 1) / bs;
  volatile int* abort_flag = &S.abort_flag;

  // ---- setup ----
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&S.kfull[i], 1);
      mbar_init(&S.kempty[i], 1);
      mbar_init(&S.vfull[i], 1);
      mbar_init(&S.vempty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.sfull[i], 1);
      mbar_init(&S.pfull[i], nact);
      mbar_init(&S.pvdone[i], 1);
    }
    mbar_init(&S.qfull, nact);
    mbar_init(&S.alldone, 1);
    S.abort_flag = 0;
    mbar_init_fence();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 5) { tmem_alloc(&S.tmem, kTmemCols); tmem_relinquish(); }
  for (int w = tid; w < words; w += kThreads) S.bits[w] = 0u;
  __syncthreads();
  // first key of a token's window
  auto window_of = [&](int64_t r) -> int {
    const int64_t e = (int64_t)a.row_pos[r] - a.local_window + 1;
    return (int)max((int64_t)0, min(e, (int64_t)ctx));
  };
  // keys [t0, t1) join the union
  auto add_range = [&](int t0, int t1) {
    t1 = min(t1, live_end);
    for (int g = t0 / GR; t0 < t1 && g * GR < t1; ++g) atomicOr(&S.bits[g >> 5], 1u << (g & 31));
  };
  for (int e = tid; e < nt * K; e += kThreads) {
    const int node = e / K;
    const int b = a.routes.idx[(r0 + node) * a.routes.row_stride + ioff + (e - node * K)];
    if (b < 0) continue;
    if (b >= nblk) { record_error(derr, DASH_DEV_BAD_BLOCK, 76, b); continue; }
    const int64_t t0 = (int64_t)b * bs;
    add_range((int)min(t0, (int64_t)ctx), (int)min(t0 + bs, (int64_t)window_of(r0 + node)));
  }
  {
    int lo = ctx;                                // the earliest window of the tile
    for (int i = lane; i < nt; i += 32) lo = min(lo, window_of(r0 + i));
    lo = __reduce_min_sync(0xffffffffu, lo);
    const int g0 = lo / GR, g1 = (live_end + GR - 1) / GR;        // [g0, g1): window and drafts
    for (int w = (g0 >> 5) + tid; w < words && w * 32 < g1; w += kThreads) {
      uint32_t m = 0xffffffffu;
      if (w * 32 < g0) m &= 0xffffffffu << (g0 & 31);
      if (w * 32 + 32 > g1) m &= 0xffffffffu >> (32 - (g1 & 31));
      atomicOr(&S.bits[w], m);
    }
  }
  __syncthreads();
  if (warp == 0) {                               // prefix sums of the words' counts
    int base = 0;
    for (int w0 = 0; w0 < words; w0 += 32) {
      const int c = w0 + lane < words ? __popc(S.bits[w0 + lane]) : 0;
      int x = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (w0 + lane < words) S.before[w0 + lane] = (uint16_t)(base + x - c);
      base += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) S.before[words] = (uint16_t)base;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  const uint32_t tO = tmem + 2 * kKeys;
  const int n_gran = S.before[words];
  const int n_tile = (n_gran + NG - 1) / NG;
  const int share = (n_tile + nsp - 1) / nsp;
  const int first = min(n_tile, split * share), tiles = min(n_tile, first + share) - first;
  const int rank0 = first * NG;

  if (warp == 4) {
    // =================== TMA producer ===================
    int it = 0;
    bool alive = true;
    for (int b0 = 0; b0 < tiles * NG && alive; b0 += 32) {
      // a lane per granule: its place in the union, its page
      const int rk = rank0 + b0 + lane;
      int tok = -1, page = (int)a.kv.num_pages;  // out of range: the box reads as zeros
      if (b0 + lane < tiles * NG && rk < n_gran) {
        int lo = 0, hi = words - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if ((int)S.before[mid] <= rk) lo = mid; else hi = mid - 1;
        }
        const int t = (lo * 32 + nth_bit(S.bits[lo], rk - S.before[lo])) * GR;
        const int64_t p = a.kv.block_table[(int64_t)s * a.kv.bt_stride + t / bs];
        if (p >= 0 && p < a.kv.num_pages) { page = (int)p; tok = t; }
        else record_error(derr, DASH_DEV_BAD_PAGE, 77, p);
      }
      const int n = min(32, tiles * NG - b0);
      for (int i = 0; i < n && alive; i += NG, ++it) {
        const int st = it % kStages;
        const uint32_t ph = (uint32_t)((it / kStages) - 1) & 1u;
        int pg[NG], tk[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          pg[g] = __shfl_sync(0xffffffffu, page, i + g);
          tk[g] = __shfl_sync(0xffffffffu, tok, i + g);
        }
        if (lane == 0) {
          if (it >= kStages && !mbar_wait(&S.kempty[st], ph, abort_flag, derr, 40)) alive = false;
          if (alive) {
            mbar_arrive_expect_tx(&S.kfull[st], kSlot);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const int row = tk[g] < 0 ? 0 : tk[g] % bs;
              tma_load_4d(S.k[st] + g * GR * 128, &tmK, &S.kfull[st], 0, row, hk, pg[g]);
              tma_load_4d(S.k[st] + 8192 + g * GR * 128, &tmK, &S.kfull[st], 64, row, hk, pg[g]);
            }
            if (it >= kStages && !mbar_wait(&S.vempty[st], ph, abort_flag, derr, 41)) alive = false;
          }
          if (alive) {
#pragma unroll
            for (int g = 0; g < NG; ++g) S.tok[st][g] = tk[g];
            mbar_arrive_expect_tx(&S.vfull[st], kSlot);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const int row = tk[g] < 0 ? 0 : tk[g] % bs;
              tma_load_4d(S.v[st] + g * GR * 128, &tmV, &S.vfull[st], 0, row, hk, pg[g]);
              tma_load_4d(S.v[st] + 8192 + g * GR * 128, &tmV, &S.vfull[st], 64, row, hk, pg[g]);
            }
          } else {
            ++it;                                // this tile's K was requested, its V was not
          }
        }
        alive = __shfl_sync(0xffffffffu, alive ? 1 : 0, 0) != 0;
      }
    }
    // never leave with bulk copies in flight (after an abort the waits run out)
    if (lane == 0) {
      volatile int no_abort = 0;
      for (int k = max(0, it - kStages); k < it; ++k) {
        mbar_wait(&S.kfull[k % kStages], (uint32_t)(k / kStages) & 1u, &no_abort, nullptr, 42);
        mbar_wait(&S.vfull[k % kStages], (uint32_t)(k / kStages) & 1u, &no_abort, nullptr, 42);
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    // =================== MMA issuer ===================
    if (lane == 0 && tiles > 0) {
      constexpr uint32_t fmt = DType<T>::fmt;
      constexpr uint32_t idesc_qk = make_idesc(fmt, 0, 0, kRows, kKeys);
      constexpr uint32_t idesc_pv = make_idesc(fmt, 0, 1, kRows, 128);
      const uint32_t sQ = smem_u32(S.q);
      bool alive = mbar_wait(&S.qfull, 0, abort_flag, derr, 50);
      auto issue_pv = [&](int j) -> bool {
        const int pb = j & 1, st = j % kStages;
        if (!mbar_wait(&S.vfull[st], (uint32_t)(j / kStages) & 1u, abort_flag, derr, 51)) return false;
        if (!mbar_wait(&S.pfull[pb], (uint32_t)(j >> 1) & 1u, abort_flag, derr, 52)) return false;
        tc_fence_after();
        const uint32_t sV = smem_u32(S.v[st]);
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          umma_ts(tO, tmem + pb * kKeys + kk * 8, sw128_desc(sV + kk * 2048, 8192, 1024), idesc_pv,
                  (j > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&S.pvdone[pb]);
        umma_commit(&S.vempty[st]);
        return true;
      };
      int it = 0;
      for (; alive && it < tiles; ++it) {
        const int st = it % kStages, sb = it & 1;
        if (!mbar_wait(&S.kfull[st], (uint32_t)(it / kStages) & 1u, abort_flag, derr, 53)) { alive = false; break; }
        // S buffer sb held P(it-2); PV(it-2) was issued before this by the same thread
        tc_fence_after();
        const uint32_t sK = smem_u32(S.k[st]);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_ss(tmem + sb * kKeys, sw128_desc(sQ + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024),
                  sw128_desc(sK + (kk >> 2) * 8192 + (kk & 3) * 32, 16, 1024), idesc_qk, kk > 0 ? 1u : 0u);
        umma_commit(&S.sfull[sb]);
        umma_commit(&S.kempty[st]);
        if (it >= 1 && !issue_pv(it - 1)) { alive = false; break; }
      }
      if (alive) issue_pv(tiles - 1);
      // every MMA is done before TMEM is given back
      umma_commit(&S.alldone);
      volatile int no_abort = 0;
      mbar_wait(&S.alldone, 0, &no_abort, nullptr, 54);
    }
    __syncwarp();
  } else if (warp < nact) {
    // =================== softmax: one thread per row ===================
    const int m = tid;                           // row of the tile = (token m / G, head m % G)
    const bool row_ok = m < nrows;
    const int node = row_ok ? m / G : 0;
    const int64_t r = r0 + node;
    const int hq = hk * G + (row_ok ? m - node * G : 0);
    {
      // a negative scale is folded into q, so that a row's largest product is
      // its largest logit
      const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
      const T* qp = reinterpret_cast<const T*>(a.qo.q) + r * a.qo.q_stride_tok + (int64_t)hq * a.qo.q_stride_head;
#pragma unroll
      for (int cc = 0; cc < 16; ++cc) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row_ok) v = __ldg(reinterpret_cast<const uint4*>(qp + cc * 8));
        v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
        *reinterpret_cast<uint4*>(S.q + (cc >> 3) * 16384 + m * 128 + (((cc & 7) ^ (m & 7)) << 4)) = v;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.qfull);
    }
    const int lstart = window_of(r);
    const uint32_t* vis = a.mask + r * a.mask_stride;
    const float sl2 = fabsf(a.scale) * kTreeLog2e;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    // granules whose terms fit the table
    const int cap = kCells / nt / NG * NG;
    int c0 = 0, c1 = 0;                          // ranks (from rank0) held by the table
    auto fill = [&](int from) {
      c0 = from;
      c1 = min(from + cap, tiles * NG);
      const int nthr = nact * 32;
      asm volatile("bar.sync 1, %0;" ::"r"(nthr) : "memory");          // the old terms have been read
      const int cells = (c1 - c0) * nt;
      int* cell_i = reinterpret_cast<int*>(S.cell);
      for (int i = m; i < cells; i += nthr) cell_i[i] = INT32_MAX;
      asm volatile("bar.sync 1, %0;" ::"r"(nthr) : "memory");
      for (int e = m; e < nt * K; e += nthr) {
        const int nd = e / K, slot = e - nd * K;
        const int b = a.routes.idx[(r0 + nd) * a.routes.row_stride + ioff + slot];
        if (b < 0 || b >= nblk) continue;
        const int64_t t0 = (int64_t)b * bs;
        const int t1 = min((int)min(t0 + bs, (int64_t)window_of(r0 + nd)), live_end);
        for (int t = (int)min(t0, (int64_t)ctx); t < t1; t += GR) {
          const int g = t / GR;
          const int rk = (int)S.before[g >> 5] + __popc(S.bits[g >> 5] & ((1u << (g & 31)) - 1u)) - rank0;
          if (rk >= c0 && rk < c1) atomicMin(cell_i + (rk - c0) * nt + nd, slot);
        }
      }
      asm volatile("bar.sync 1, %0;" ::"r"(nthr) : "memory");
      for (int i = m; i < cells; i += nthr) {
        const int slot = cell_i[i];
        float t = -INFINITY;
        if (slot != INT32_MAX)
          t = a.routes.bias
                  ? a.routes.bias[(r0 + i % nt) * a.routes.row_stride + ioff + slot] * kTreeLog2e
                  : 0.0f;
        S.cell[i] = t;
      }
      asm volatile("bar.sync 1, %0;" ::"r"(nthr) : "memory");
    };
    float m_run = -INFINITY, l_run = 0.0f;
    bool alive = true;
    for (int it = 0; it < tiles; ++it) {
      if (it * NG >= c1) fill(it * NG);
      if (!alive) continue;                      // after an abort: only the table's barriers
      const int st = it % kStages, sb = it & 1;
      if (!mbar_wait_warp(&S.vfull[st], (uint32_t)(it / kStages) & 1u, abort_flag, derr, 60)) { alive = false; continue; }
      int t0[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) t0[g] = S.tok[st][g];
      // V rows behind the last drafted token: P = 0 must not meet a NaN
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        if (t0[g] >= 0 && t0[g] + GR > end) {
          const int q0 = max(0, end - t0[g]);
          for (int e = m; e < (GR - q0) * 16; e += nact * 32) {
            const int row = g * GR + q0 + e / 16, ch = e % 16;
            *reinterpret_cast<uint4*>(S.v[st] + (ch >> 3) * 8192 + row * 128 + ((ch & 7) << 4)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
      }
      if (!mbar_wait_warp(&S.sfull[sb], (uint32_t)(it >> 1) & 1u, abort_flag, derr, 61)) { alive = false; continue; }
      tc_fence_after();
      const uint32_t tS = tmem + sb * kKeys + lane_base;
      float x[kKeys];
      tmem_ld32f(tS, x);
      tmem_ld32f(tS + 32, x + 32);
      // additive term of each granule for this row; pure: one term for all GR keys
      float add[NG];
      bool pure = true, none = true;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        add[g] = -INFINITY;
        if (t0[g] >= 0 && row_ok) {
          const bool remote = t0[g] < lstart;
          if (remote) add[g] = S.cell[(it * NG + g - c0) * nt + node];
          else if (t0[g] + GR <= ctx) add[g] = 0.0f;
          const bool p = remote ? t0[g] + GR <= lstart : t0[g] + GR <= ctx;
          pure &= p;
          none &= p && add[g] == -INFINITY;
        }
      }
      tmem_ld_wait();
      uint32_t pk[kKeys / 2];
      if (__all_sync(0xffffffffu, none)) {
        // no row of this warp attends the tile
#pragma unroll
        for (int e = 0; e < kKeys / 2; ++e) pk[e] = 0u;
      } else {
        const bool all_pure = __all_sync(0xffffffffu, pure);
        float mx = -INFINITY;
        if (all_pure) {
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float h = -INFINITY;
#pragma unroll
            for (int c = 0; c < GR; ++c) h = fmaxf(h, x[g * GR + c]);
            mx = fmaxf(mx, fmaf(h, sl2, add[g]));                       // sl2 >= 0
          }
        } else {
          // key by key: remote keys take the granule's term, window and
          // visible drafted keys none, all others -inf
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            uint64_t on = 0;                     // columns attended without a term
            int rem = 0;                         // columns [0, rem) are remote
            if (t0[g] >= 0 && row_ok) {
              rem = min(GR, max(0, lstart - t0[g]));
              const int loc = min(GR, max(0, ctx - t0[g]));            // columns [rem, loc) are the window
              const uint64_t below = loc >= 64 ? ~0ull : (1ull << loc) - 1ull;
              on = below & (rem >= 64 ? 0ull : ~0ull << rem);
              if (loc < GR) {
                const int v0 = t0[g] + loc - ctx;                       // drafted token of column loc
                uint64_t bits = 0;
#pragma unroll
                for (int w = 0; w < 3; ++w) {
                  const int wi = (v0 >> 5) + w;
                  if (wi < a.mask_words && wi * 32 < total_n) {
                    uint32_t mw = vis[wi];
                    if (total_n - wi * 32 < 32) mw &= (1u << (total_n - wi * 32)) - 1u;
                    const int sh = wi * 32 - v0;                        // column of the word's first token - loc
                    if (sh >= 0) { if (sh < 64) bits |= (uint64_t)mw << sh; }
                    else bits |= (uint64_t)(mw >> -sh);
                  }
                }
                on |= bits << loc;
              }
            }
#pragma unroll
            for (int c = 0; c < GR; ++c) {
              const float y = fmaf(x[g * GR + c], sl2, c < rem ? add[g] : 0.0f);
              x[g * GR + c] = (c < rem || ((on >> c) & 1ull)) ? y : -INFINITY;
              mx = fmaxf(mx, x[g * GR + c]);
            }
          }
        }
        // running maximum; O follows it only when it grew by more than 2^kGrow
        const bool grow = mx > m_run + kGrow;
        const bool scale_o = grow && m_run != -INFINITY;
        if (__any_sync(0xffffffffu, scale_o)) {
          const float f = scale_o ? fast_exp2(m_run - mx) : 1.0f;
          if (it > 0) {
            if (!mbar_wait_warp(&S.pvdone[(it - 1) & 1], (uint32_t)((it - 1) >> 1) & 1u, abort_flag, derr, 62)) {
              alive = false;
              continue;
            }
            tc_fence_after();
#pragma unroll 1
            for (int q4 = 0; q4 < 4; ++q4) {
              uint32_t o[32];
              tmem_ld32(tO + q4 * 32 + lane_base, o);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
              tmem_st32(tO + q4 * 32 + lane_base, o);
            }
            tmem_st_wait();
          }
          l_run *= f;
        }
        if (grow) m_run = mx;
        const float mu = m_run == -INFINITY ? 0.0f : m_run;
        uint64_t ls = f2_pack(0.0f, 0.0f);
        if (all_pure) {
          const uint64_t sl = f2_pack(sl2, sl2);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint64_t ad = f2_pack(add[g] - mu, add[g] - mu);
#pragma unroll
            for (int c = 0; c < GR; c += 2) {
              float y0, y1;
              f2_unpack(ffma2(f2_pack(x[g * GR + c], x[g * GR + c + 1]), sl, ad), y0, y1);
              const float p0 = fast_exp2(y0), p1 = fast_exp2(y1);
              ls = fadd2(ls, f2_pack(p0, p1));
              pk[(g * GR + c) >> 1] = pack2(p0, p1, (T*)nullptr);
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < kKeys; c += 2) {
            const float p0 = fast_exp2(x[c] - mu), p1 = fast_exp2(x[c + 1] - mu);
            ls = fadd2(ls, f2_pack(p0, p1));
            pk[c >> 1] = pack2(p0, p1, (T*)nullptr);
          }
        }
        float l0, l1;
        f2_unpack(ls, l0, l1);
        l_run += l0 + l1;
      }
      tmem_st32(tS, pk);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.pfull[sb]);
    }
    // ---- O, maximum and sum into shared memory (the K and V slots are free) ----
    if (tiles > 0 && alive)
      alive = mbar_wait_warp(&S.pvdone[(tiles - 1) & 1], (uint32_t)((tiles - 1) >> 1) & 1u, abort_flag, derr, 63);
    tc_fence_after();
    if (tiles > 0) {
#pragma unroll 1
      for (int q4 = 0; q4 < 4; ++q4) {
        uint32_t o[32];
        tmem_ld32(tO + q4 * 32 + lane_base, o);
        tmem_ld_wait();
#pragma unroll
        for (int v = 0; v < 8; ++v)
          *reinterpret_cast<uint4*>(S.k[0] + m * 512 + (((q4 * 8 + v) ^ (m & 7)) << 4)) =
              make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
      }
    }
    S.m[m] = m_run;
    S.l[m] = tiles > 0 ? l_run : -1.0f;          // -1: this CTA had no tile
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, kTmemCols);
  cluster.sync();
  // ---- join: row m by CTA m % nsp, a warp per row, lane = 4 dims ----
  for (int m = split + nsp * warp; m < nrows; m += nsp * (kThreads / 32)) {
    const int node = m / G;
    const int64_t r = r0 + node;
    const int hq = hk * G + m - node * G;
    float M = -INFINITY;
    float mk = -INFINITY, lk = -1.0f;            // lane k holds CTA k's
    if (lane < nsp) {
      mk = *cluster.map_shared_rank(&S.m[m], lane);
      lk = *cluster.map_shared_rank(&S.l[m], lane);
    }
    M = mk;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    M = __shfl_sync(0xffffffffu, M, 0);
    float L = 0.0f;
    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < nsp; ++k) {
      const float m1 = __shfl_sync(0xffffffffu, mk, k), l1 = __shfl_sync(0xffffffffu, lk, k);
      if (l1 == -1.0f) continue;
      const float w = m1 == -INFINITY ? 0.0f : fast_exp2(m1 - M);
      const float4 o =
          *reinterpret_cast<const float4*>(cluster.map_shared_rank(&S.k[0][0], k) + m * 512 + ((lane ^ (m & 7)) << 4));
      L += l1 * w;
      O.x += o.x * w; O.y += o.y * w; O.z += o.z * w; O.w += o.w * w;
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    // x * 0 is 0 for a finite x only
    const bool fine = (O.x + O.y + O.z + O.w) * 0.0f + L * 0.0f == 0.0f;
    if (!__all_sync(0xffffffffu, fine)) {
      float ms, ls, os[16];
      tree_row_attend<T>(a, sq, s, r, hq, ms, ls, os);
      tree_row_store<T>(a, r, hq, ms, ls, os);
      continue;
    }
    T* op = reinterpret_cast<T*>(a.qo.out) + r * a.qo.o_stride_tok + (int64_t)hq * a.qo.o_stride_head + lane * 4;
    *reinterpret_cast<uint2*>(op) =
        make_uint2(pack2(O.x * inv, O.y * inv, (T*)nullptr), pack2(O.z * inv, O.w * inv, (T*)nullptr));
    if (lane == 0 && a.qo.lse)
      a.qo.lse[r * a.qo.lse_stride_tok + (int64_t)hq * a.qo.lse_stride_head] =
          L > 0.0f ? (M + log2f(L)) * kTreeLn2 : -INFINITY;
  }
  cluster.sync();                                // no CTA leaves while another reads its part
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static PFN_cuTensorMapEncodeTiled_v12000 tree_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

static int granule_of(int bs) { return bs == 16 || bs == 32 ? bs : bs % 64 == 0 && bs <= 256 ? 64 : 0; }

// Block sizes that a 64-key tile is made of, up to 128 query heads per kv head,
// a table whose granules fit the bit set, layouts that TMA takes.
bool tree_tc_supported(const DashTreeAttnArgs& a) {
  const int gr = granule_of(a.block_size);
  return gr && a.qo.n_heads / a.kv.n_kv_heads <= kRows &&
         (int64_t)a.bt_width * a.block_size <= (int64_t)kMaxWords * 32 * gr && a.kv.stride_tok > 0 &&
         a.kv.stride_head > 0 && a.kv.stride_seq > 0 && tree_encode_fn() != nullptr;
}

static int page_map(CUtensorMap* map, const void* base, const DashTreeAttnArgs& a, int gr) {
  cuuint64_t dims[4] = {128, (cuuint64_t)a.block_size, (cuuint64_t)a.kv.n_kv_heads, (cuuint64_t)a.kv.num_pages};
  cuuint64_t strides[3] = {(cuuint64_t)a.kv.stride_tok * 2, (cuuint64_t)a.kv.stride_head * 2,
                           (cuuint64_t)a.kv.stride_seq * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)gr, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = tree_encode_fn()(
      map, a.kv.dtype == DASH_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
      const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(DASH_ERR_CUDA, "cuTensorMapEncodeTiled (tree K/V) failed (%d)", (int)r);
  return DASH_OK;
}

// CTAs per sequence and kv head: (whole waves of CTAs, two per SM) x (tiles of a
// CTA + setup and join, worth about 3 tiles).  The number of tiles is not known
// here; its upper bound is.
static int tree_splits(const DashTreeAttnArgs& a, int64_t units, int gr) {
  if (a.num_splits) return a.num_splits;
  const int64_t per = kRows / (a.qo.n_heads / a.kv.n_kv_heads);
  const int64_t nodes = a.seqs.max_q_len < per ? a.seqs.max_q_len : per;
  int64_t gran = nodes * a.routes.K * (a.block_size / gr) + (a.local_window + nodes) / gr + 2;
  const int64_t most = (int64_t)a.bt_width * a.block_size / gr;
  if (gran > most) gran = most;
  const int64_t tiles = (gran * gr + kKeys - 1) / kKeys;
  int best = 1;
  int64_t cost = INT64_MAX;
  for (int sp = 1; sp <= 8 && sp <= tiles; ++sp) {
    const int64_t waves = (units * sp + 295) / 296, c = waves * ((tiles + sp - 1) / sp + 3);
    if (c < cost) { cost = c; best = sp; }
  }
  return best;
}

template <typename T, int GR>
static int launch_tc(const DashTreeAttnArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  const int per = kRows / (a.qo.n_heads / a.kv.n_kv_heads);
  const int n_tiles = (a.seqs.max_q_len + per - 1) / per;
  const int64_t units = (int64_t)a.seqs.n_seq * a.kv.n_kv_heads * n_tiles;
  const int sp = tree_splits(a, units, GR);
  if (units * sp > INT32_MAX) return set_error(DASH_ERR_UNSUPPORTED, "too many sequences x kv heads");
  const int smem = (int)sizeof(TreeSmem) + 1024;
  auto kernel = tree_tc_kernel<T, GR>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * sp));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)sp;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, mk, mv, a, n_tiles);
  }
  if (e != cudaSuccess) return set_error(DASH_ERR_CUDA, "tree_tc_kernel launch failed: %s", cudaGetErrorString(e));
  count_launch();
  return check_launch("tree_tc_kernel");
}

template <typename T>
static int launch_tc_gr(const DashTreeAttnArgs& a, cudaStream_t st) {
  const int gr = granule_of(a.block_size);
  CUtensorMap mk, mv;
  int rc = page_map(&mk, a.kv.k, a, gr);
  if (rc == DASH_OK) rc = page_map(&mv, a.kv.v, a, gr);
  if (rc != DASH_OK) return rc;
  if (gr == 16) return launch_tc<T, 16>(a, mk, mv, st);
  if (gr == 32) return launch_tc<T, 32>(a, mk, mv, st);
  return launch_tc<T, 64>(a, mk, mv, st);
}

int launch_tree_tc(const DashTreeAttnArgs& a, cudaStream_t st) {
  return a.kv.dtype == DASH_DTYPE_BF16 ? launch_tc_gr<__nv_bfloat16>(a, st) : launch_tc_gr<__half>(a, st);
}

}  // namespace dash
