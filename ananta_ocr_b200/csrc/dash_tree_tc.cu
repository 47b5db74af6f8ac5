// dash_tree_tc.cu -- draft-tree attention on the sm_100a tensor cores.
//
// Work unit: up to 128 (drafted token, query head) rows of one sequence and kv
// head, split over a cluster of 1..16 CTAs.  The keys that any row attends --
// the union of the rows' routed blocks, their windows and the drafted tokens --
// are cut into granules of GR tokens (GR = block size, 64 at most); a tile of 64
// keys is 64 / GR granules of the union in ascending order, and each CTA of the
// cluster takes a contiguous part of the tiles.  Every key of the union crosses
// the memory bus once per kv head, whatever the number of drafted tokens, which is
// what bounds the kernel: 32 KB of K and V per tile against ~0.5 k cycles of
// tensor work (M = 128 rows, padded) and ~0.6 k of softmax per SM sub-partition.
//
//   setup             union bit set and its prefix sums in shared memory, while Q
//                     arrives by cp.async
//   warp 4  TMA       block table -> page boxes {64 dims, GR tokens} of K and V
//                     (128-byte swizzle), K and V in rings of their own (16 KB per
//                     slot): a K slot is free after Q K^T, a V slot after P V
//   warp 5  MMA       S = Q K^T (M 128, N 64, two TMEM buffers), O += P V (N 128, P
//                     from TMEM)
//   warps 0-3 softmax one thread per row; warps without a row sleep.  The additive
//                     terms of the routed granules lie in a [granule][token]
//                     table (of a repeated id the lowest slot's), refilled when
//                     a part outgrows it
//
// Units of up to 32 rows keep 8 KB of Q and three K and V slots, of up to 64 rows 16 KB,
// three and two, larger ones 32 KB and two (the rows of Q's operand tile that do not exist are whatever lies
// behind them: they make rows of S that nobody reads).  Either way two CTAs fit an SM
// (256 TMEM columns each), and their phases interleave.  At the end the CTAs leave O,
// the running maximum and the sum in their shared memory and each joins its share
// of the rows over the cluster (no workspace, no atomics, fixed order); a CTA
// that holds a unit alone writes it from its registers.
//
// A CTA lives for some 20 us and runs most of its code once, so instruction fetches
// count: loops that are not in the tiles' path stay rolled (unrolled, warps waited
// 5 us per CTA for instructions).
//
// Measured (CUDA graph, bf16, window 4 blocks): 32 sequences of one token on 27,556 (block
// 64, K 32, 10 kv heads) 78 us, 4.8 TB/s of the 378 MB that the union needs; 16 trees
// of 16 47 us (4.0 TB/s), 8 of 17 on blocks of 32 20.5 us, one of 8 14.5 us (launch, set-up
// and join: 10 us of fixed cost); four of 64 with four heads per kv head 33 us.
//
// A masked key has P = 0, and 0 * v is 0 only for finite v.  V rows behind the last
// drafted token are zeroed; a row whose joined output is not finite for any
// other reason (a bad value in a key that some other row attends, or in its own)
// is computed again from its own keys only (tree_row_attend), so no row's
// result depends on keys that it does not attend, except in its last bits: there
// the weights are not rounded to the caches' type.  Computed again is also a row
// that has no key but in blocks of the lowest biases (below -1e30, where a bias
// times log2(e) may leave the type's range and the logit is lost beside it).
#include <cooperative_groups.h>
#include <cudaTypedefs.h>
#include <cfloat>
#include "dash_tree.cuh"

namespace cg = cooperative_groups;

namespace dash {
namespace {

constexpr int kRows = 128;                       // M of both MMAs
constexpr int kKeys = 64;                        // N of Q K^T, K of P V
constexpr int kThreads = 192;
constexpr int kSlot = 16384;                     // one tile of K or of V: 2 x [64 x 128 B]
constexpr int kMaxCluster = 16;
constexpr int kMaxWords = 256;                   // 8192 granules of a sequence
constexpr uint32_t kTmemCols = 256;              // S0 | S1 | O
constexpr float kGrow = 8.0f;                    // O is rescaled when a row's maximum grows by 2^8
constexpr float kFar = -1e30f;                   // below it a row's maximum is one of the lowest biases'

// QR: rows of Q that are kept (32, 64 or 128)
template <int QR>
struct TreeSmem {
  static constexpr int kKSlots = QR <= 64 ? 3 : 2, kVSlots = QR == 32 ? 3 : 2;
  static constexpr int kCells = QR == 32 ? 980 : QR == 64 ? 2900 : 2800;      // additive terms held at a time
  static constexpr int kSlots = 1024;            // routed slots held
  uint8_t q[2 * QR * 128];                       // two halves of 64 dims, swizzled
  uint8_t k[kKSlots][kSlot];                     // receives O (QR x 512 B) at the end
  uint8_t v[kVSlots][kSlot];
  float cell[kCells];
  uint16_t slot[kSlots];                         // (first granule << 3) | granules
  uint32_t bits[kMaxWords];
  uint16_t before[kMaxWords + 2];
  int tok[8][4];                                 // first token of the tile's granules, -1 = none (K runs < 8 tiles ahead)
  float m[QR], l[QR];
  uint64_t kfull[kKSlots], kempty[kKSlots], vfull[kVSlots], vempty[kVSlots];
  uint64_t sfull[2], pfull[2], pvdone[2], qfull, alldone;
  uint32_t tmem;
  int abort_flag;
};
template <int QR>
constexpr bool fits() {
  using S = TreeSmem<QR>;
  // two CTAs per SM; O fits the K and V slots; Q's operand tile stays inside
  return sizeof(S) + 1024 <= 233472 / 2 - 1024 && QR * 512 <= (S::kKSlots + S::kVSlots) * kSlot &&
         QR * 128 + kRows * 128 <= (int)sizeof(S::q) + S::kKSlots * kSlot && offsetof(S, k) == sizeof(S::q) &&
         offsetof(S, v) == offsetof(S, k) + sizeof(S::k);
}
static_assert(fits<32>() && fits<64>() && fits<128>(), "shared memory of a CTA");

// Row m of a unit from its own keys only (the whole warp).  Its query comes from the
// operand tile sq_q (halves of `half` bytes), because the output may lie on q.
template <typename T>
__device__ __noinline__ void redo_row(const DashTreeAttnArgs& a, TreeSeq sq, int s, int64_t r0, int m, int G,
                                      int hk, const uint8_t* sq_q, int half) {
  const int node = m / G, hq = hk * G + m - node * G;
  const int c0 = 2 * (threadIdx.x & 7), c1 = c0 + 1;             // the lane's 16-byte pieces
  auto piece = [&](int c) {
    return *reinterpret_cast<const uint4*>(sq_q + (c >> 3) * half + m * 128 + (((c & 7) ^ (m & 7)) << 4));
  };
  float q[16], ms, ls, os[16];
  tree_load_q<T>(piece(c0), piece(c1), q);
  tree_row_attend<T>(a, sq, s, r0 + node, hq, q, fabsf(a.scale), ms, ls, os);     // (its sign is in the tile)
  tree_row_store<T>(a, r0 + node, hq, ms, ls, os);
}

// the j-th set bit of w (j < popc(w))
__device__ __forceinline__ int nth_bit(uint32_t w, int j) { return (int)__fns(w, 0, j + 1); }

// Bounded wait (see mbar_wait), small enough to stand in many places: a few polls,
// then out of line.
__device__ __noinline__ bool tree_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, DeviceError* err,
                                            int where) {
  return mbar_wait(bar, parity, abort_flag, err, where);
}
__device__ __forceinline__ bool tree_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, DeviceError* err,
                                          int where) {
#pragma unroll 1
  for (int i = 0; i < 8; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return tree_wait_long(bar, parity, abort_flag, err, where);
}
__device__ __forceinline__ bool tree_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                               DeviceError* err, int where) {
  return __all_sync(0xffffffffu, tree_wait(bar, parity, abort_flag, err, where));
}

// whether the phase is complete, without waiting
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ void tmem_ld16f(uint32_t taddr, float (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16f(uint32_t taddr, const float (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
      "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

}  // namespace

template <typename T, int GR, int QR>
__global__ void __launch_bounds__(kThreads, 2)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ DashTreeAttnArgs a, int n_tiles_seq, int unit0, bool more) {
  constexpr int NG = kKeys / GR;                 // granules per tile
  using Smem = TreeSmem<QR>;
  constexpr int kKSlots = Smem::kKSlots, kVSlots = Smem::kVSlots;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& S = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  cg::cluster_group cluster = cg::this_cluster();
  const int nsp = (int)cluster.num_blocks(), split = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int u = unit0 + blockIdx.x / nsp;
  const int tile_i = u % n_tiles_seq;
  u /= n_tiles_seq;
  const int hk = u % a.kv.n_kv_heads, s = u / a.kv.n_kv_heads;
  const int H = a.qo.n_heads, G = H / a.kv.n_kv_heads, bs = a.block_size;
  const int per_tile = kRows / G;                // tokens of a tile
  TreeSeq sq = tree_seq(a.seqs.q_start, a.ctx_len, a.seqs.q_len_fixed, a.seqs.max_q_len, s);
  const int node0 = tile_i * per_tile;
  const int nt = min(per_tile, sq.n - node0);    // this tile's tokens
  // Of two launches the second takes the slots that the first leaves, as soon as it
  // leaves them; it ends after the first, so that what follows sees both.
  if (more) asm volatile("griddepcontrol.launch_dependents;");
  auto after_first = [&]() {
    if (unit0 > 0) asm volatile("griddepcontrol.wait;" ::: "memory");
  };
  if (nt <= 0) {                                 // the whole cluster leaves
    after_first();
    return;
  }
  const int total_n = sq.n;
  const int64_t r0 = sq.row0 + node0;            // packed row of the tile's first token
  const int nrows = nt * G, nact = (nrows + 31) >> 5;
  const int nih = a.routes.n_index_heads > 0 ? a.routes.n_index_heads : 1;
  const int K = a.routes.K;
  const int64_t rbase = r0 * a.routes.row_stride + (int64_t)((hk * G) / (H / nih)) * a.routes.ihead_stride;
  DeviceError* derr = a.device_error;
  const int ctx = sq.ctx, end = ctx + total_n;
  // tokens behind the table's last column do not exist
  const int64_t room = (int64_t)a.bt_width * bs;
  const int live_end = (int)min((int64_t)end, room);
  const int words = min(kMaxWords, (live_end + 32 * GR - 1) / (32 * GR));
  if (live_end < end && tid == 0 && hk == 0 && split == 0) record_error(derr, DASH_DEV_BAD_PAGE, 75, a.bt_width);
  const int nblk = (end + bs - 1) / bs;
  volatile int* abort_flag = &S.abort_flag;

  // first key of a row's window
  auto window_of = [&](int64_t r) -> int {
    const int64_t e = (int64_t)__ldg(a.row_pos + r) - a.local_window + 1;
    return (int)max((int64_t)0, min(e, (int64_t)ctx));
  };
  // entry e = (token, slot of its list), lists padded to a power of two
  const int pad = K > 1 ? 32 - __clz(K - 1) : 0;
  const int entries = K > 0 ? nt << pad : 0;
  // remote granules of block b for a row at position pos: (first << 3) | count (13 and 3 bits)
  auto remote = [&](int b, int pos) -> uint32_t {
    if (b >= nblk) record_error(derr, DASH_DEV_BAD_BLOCK, 76, b);
    const int64_t e = (int64_t)pos - a.local_window + 1;
    const int edge = (int)max((int64_t)0, min(e, (int64_t)min(ctx, live_end)));
    const int64_t t0 = (int64_t)b * bs, t1 = min(t0 + bs, (int64_t)edge);
    return b >= 0 && t1 > t0 ? (uint32_t)(t0 / GR) << 3 | (uint32_t)((t1 - t0 + GR - 1) / GR) : 0u;
  };
  // the same for entry e, from memory
  auto remote_of = [&](int e) -> uint32_t {
    const int node = e >> pad, slot = e & ((1 << pad) - 1);
    return slot < K ? remote(__ldg(a.routes.idx + rbase + (int64_t)node * a.routes.row_stride + slot),
                             __ldg(a.row_pos + r0 + node))
                    : 0u;
  };

  // ---- setup ----
  if (warp == 5) {
    tmem_alloc(&S.tmem, kTmemCols);
    tmem_relinquish();
    if (lane < kKSlots) {
      mbar_init(&S.kfull[lane], 1);
      mbar_init(&S.kempty[lane], 1);
    }
    if (lane < kVSlots) {
      mbar_init(&S.vfull[lane], 1);
      mbar_init(&S.vempty[lane], 1);
    }
    if (lane < 2) {
      mbar_init(&S.sfull[lane], 1);
      mbar_init(&S.pfull[lane], nact);
      mbar_init(&S.pvdone[lane], 1);
    }
    if (lane == 0) {
      mbar_init(&S.qfull, 2);
      mbar_init(&S.alldone, 1);
      S.abort_flag = 0;
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
    mbar_init_fence();
  }
  if (warp >= 4) {
    // the table's row on its way to the L1, for the producer
    for (int b = (tid - kRows) * 32; b < min(a.bt_width, nblk); b += (kThreads - kRows) * 32)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(a.kv.block_table + (int64_t)s * a.kv.bt_stride + b));
    // Q (rows of the operand tile beyond the unit's stay as they are)
#pragma unroll 4
    for (int c = tid - kRows; c < nrows * 16; c += kThreads - kRows) {
      const int m = c >> 4, cc = c & 15, node = m / G;
      const T* src = reinterpret_cast<const T*>(a.qo.q) + (r0 + node) * a.qo.q_stride_tok +
                     (int64_t)(hk * G + m - node * G) * a.qo.q_stride_head + cc * 8;
      const uint32_t dst = smem_u32(S.q + (cc >> 3) * (QR * 128) + m * 128 + (((cc & 7) ^ (m & 7)) << 4));
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    }
  } else {
    // ---- the union ----
    const int first_key = tid < nt ? window_of(r0 + tid) : ctx;
    for (int w = tid; w < kMaxWords; w += kRows) S.bits[w] = 0u;
    asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll 1
    for (int e0 = tid; e0 < entries; e0 += 4 * kRows) {
      int b[4], pos[4];                          // the loads of four entries at once
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i * kRows, node = e >> pad, slot = e & ((1 << pad) - 1);
        b[i] = -1;
        pos[i] = 0;
        if (e < entries && slot < K) {
          const int64_t at = rbase + (int64_t)node * a.routes.row_stride + slot;
          b[i] = __ldg(a.routes.idx + at);
          pos[i] = __ldg(a.row_pos + r0 + node);
          // the biases are read next, by the same threads
          if (a.routes.bias) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.routes.bias + at));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i * kRows;
        const uint32_t v = remote(b[i], pos[i]);
        if (e < Smem::kSlots) S.slot[e] = (uint16_t)v;
        // (tokens of a tree name the same blocks: a set bit needs no atomic)
        for (uint32_t g = v >> 3, g1 = g + (v & 7u); g < g1; ++g)
          if (!((*(volatile uint32_t*)&S.bits[g >> 5] >> (g & 31)) & 1u)) atomicOr(&S.bits[g >> 5], 1u << (g & 31));
      }
    }
    // the windows of the warp's tokens and the drafts: granules [g0, g1)
    const int g0 = __reduce_min_sync(0xffffffffu, first_key) / GR, g1 = (live_end + GR - 1) / GR;
    for (int w = (g0 >> 5) + lane; w * 32 < g1; w += 32) {
      uint32_t m = 0xffffffffu;
      if (w * 32 < g0) m &= 0xffffffffu << (g0 & 31);
      if (w * 32 + 32 > g1) m &= 0xffffffffu >> (32 - (g1 & 31));
      atomicOr(&S.bits[w], m);
    }
  }
  __syncthreads();
  if (warp == 0) {                               // prefix sums of the words' counts
    int base = 0;
#pragma unroll 1
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
  uint32_t redo = 0;                             // rows of this warp to be computed again

  if (warp >= 4) {
    // Q has come (requested at the start)
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (a.scale < 0.0f) {
      // a negative scale is folded into q, so that a row's largest product is
      // its largest logit
#pragma unroll 1
      for (int c = tid - kRows; c < nrows * 16; c += kThreads - kRows) {
        const int m = c >> 4, cc = c & 15;
        uint4* p = reinterpret_cast<uint4*>(S.q + (cc >> 3) * (QR * 128) + m * 128 + (((cc & 7) ^ (m & 7)) << 4));
        uint4 v = *p;
        v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u;
        *p = v;
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&S.qfull);
  }
  if (warp == 4) {
    // =================== TMA producer ===================
    // K runs a tile ahead of V, so that a V slot that is still read does not keep
    // the next K from being requested.
    int kn = 0, vn = 0;                          // tiles requested
    int page = 0, tok = 0;                       // a lane's granule of the current 32
    int vpg[NG], vtk[NG];                        // the tile whose V is next
    bool alive = true;
#pragma unroll 1
    for (int it = 0; it <= tiles && alive; ++it) {
      int pg[NG], tk[NG];
      if (it < tiles) {
        const int at = it * NG & 31;
        if (at == 0) {
          // a lane per granule: its place in the union, its page
          const int rk = rank0 + it * NG + lane;
          tok = -1;
          page = (int)a.kv.num_pages;            // out of range: the box reads as zeros
          if (it * NG + lane < tiles * NG && rk < n_gran) {
            int lo = 0, hi = words - 1;
            while (lo < hi) {
              const int mid = (lo + hi + 1) >> 1;
              if ((int)S.before[mid] <= rk) lo = mid; else hi = mid - 1;
            }
            const int t = (lo * 32 + nth_bit(S.bits[lo], rk - S.before[lo])) * GR;
            const int64_t p = __ldg(a.kv.block_table + (int64_t)s * a.kv.bt_stride + t / bs);
            if (p >= 0 && p < a.kv.num_pages) { page = (int)p; tok = t; }
            else record_error(derr, DASH_DEV_BAD_PAGE, 77, p);
          }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          pg[g] = __shfl_sync(0xffffffffu, page, at + g);
          tk[g] = __shfl_sync(0xffffffffu, tok, at + g);
        }
        if (lane == 0) {
          const int st = it % kKSlots;
          if (it >= kKSlots && !tree_wait(&S.kempty[st], (uint32_t)((it / kKSlots) - 1) & 1u, abort_flag, derr, 40)) {
            alive = false;
          } else {
#pragma unroll
            for (int g = 0; g < NG; ++g) S.tok[it & 7][g] = tk[g];
            mbar_arrive_expect_tx(&S.kfull[st], kSlot);
            ++kn;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const int row = tk[g] < 0 ? 0 : tk[g] % bs;
              tma_load_4d(S.k[st] + g * GR * 128, &tmK, &S.kfull[st], 0, row, hk, pg[g]);
              tma_load_4d(S.k[st] + 8192 + g * GR * 128, &tmK, &S.kfull[st], 64, row, hk, pg[g]);
            }
          }
        }
      }
      if (it > 0 && lane == 0 && alive) {
        const int j = it - 1, st = j % kVSlots;
        if (j >= kVSlots && !tree_wait(&S.vempty[st], (uint32_t)((j / kVSlots) - 1) & 1u, abort_flag, derr, 41)) {
          alive = false;
        } else {
          mbar_arrive_expect_tx(&S.vfull[st], kSlot);
          ++vn;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const int row = vtk[g] < 0 ? 0 : vtk[g] % bs;
            tma_load_4d(S.v[st] + g * GR * 128, &tmV, &S.vfull[st], 0, row, hk, vpg[g]);
            tma_load_4d(S.v[st] + 8192 + g * GR * 128, &tmV, &S.vfull[st], 64, row, hk, vpg[g]);
          }
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) { vpg[g] = pg[g]; vtk[g] = tk[g]; }
      alive = __shfl_sync(0xffffffffu, alive ? 1 : 0, 0) != 0;
    }
    // never leave with bulk copies in flight (after an abort the waits run out)
    if (lane == 0) {
      volatile int no_abort = 0;
#pragma unroll 1
      for (int k = max(0, kn - kKSlots); k < kn; ++k)
        tree_wait(&S.kfull[k % kKSlots], (uint32_t)(k / kKSlots) & 1u, &no_abort, nullptr, 42);
#pragma unroll 1
      for (int k = max(0, vn - kVSlots); k < vn; ++k)
        tree_wait(&S.vfull[k % kVSlots], (uint32_t)(k / kVSlots) & 1u, &no_abort, nullptr, 42);
    }
    __syncwarp();
  } else if (warp == 5) {
    // =================== MMA issuer ===================
    if (lane == 0 && tiles > 0) {
      constexpr uint32_t fmt = DType<T>::fmt;
      constexpr uint32_t idesc_qk = make_idesc(fmt, 0, 0, kRows, kKeys);
      constexpr uint32_t idesc_pv = make_idesc(fmt, 0, 1, kRows, 128);
      const uint32_t sQ = smem_u32(S.q);
      // S(qk) = Q K^T and O += P(pv) V are issued as their operands come, whichever is
      // first: a K tile that is late does not hold back the P V that frees a V slot.
      // S buffer qk & 1 held P(qk - 2), whose P V was issued before by this thread.
      int qk = 0, pv = tree_wait(&S.qfull, 0, abort_flag, derr, 50) ? 0 : tiles;
      uint32_t idle = 0;
      uint64_t since = 0;
#pragma unroll 1
      while (pv < tiles) {
        bool did = false;
        if (pv < qk && mbar_test(&S.pfull[pv & 1], (uint32_t)(pv >> 1) & 1u) &&
            mbar_test(&S.vfull[pv % kVSlots], (uint32_t)(pv / kVSlots) & 1u)) {
          tc_fence_after();
          const uint32_t sV = smem_u32(S.v[pv % kVSlots]);
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            umma_ts(tO, tmem + (pv & 1) * kKeys + kk * 8, sw128_desc(sV + kk * 2048, 8192, 1024), idesc_pv,
                    (pv > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&S.pvdone[pv & 1]);
          umma_commit(&S.vempty[pv % kVSlots]);
          ++pv;
          did = true;
        }
        if (qk < tiles && qk <= pv + 1 && mbar_test(&S.kfull[qk % kKSlots], (uint32_t)(qk / kKSlots) & 1u)) {
          tc_fence_after();
          const uint32_t sK = smem_u32(S.k[qk % kKSlots]);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ss(tmem + (qk & 1) * kKeys, sw128_desc(sQ + (kk >> 2) * (QR * 128) + (kk & 3) * 32, 16, 1024),
                    sw128_desc(sK + (kk >> 2) * 8192 + (kk & 3) * 32, 16, 1024), idesc_qk, kk > 0 ? 1u : 0u);
          umma_commit(&S.sfull[qk & 1]);
          umma_commit(&S.kempty[qk % kKSlots]);
          ++qk;
          did = true;
        }
        if (did) {
          idle = 0;
        } else if ((++idle & 255u) == 0) {       // the wait is bounded as all others are
          if (idle == 256u) since = globaltimer_ns();
          if (*abort_flag) break;
          if (globaltimer_ns() - since > 2000000000ull) {
            *abort_flag = 1;
            record_error(derr, DASH_DEV_TIMEOUT, 51, qk);
            break;
          }
        }
      }
      // every MMA is done before TMEM is given back
      umma_commit(&S.alldone);
      volatile int no_abort = 0;
      tree_wait(&S.alldone, 0, &no_abort, nullptr, 54);
    }
    __syncwarp();
  } else {
    // =================== softmax: one thread per row ===================
    const int m = tid;                           // row of the unit = (token m / G, head m % G)
    const bool row_ok = m < nrows, warp_on = warp < nact;
    const int node = row_ok ? m / G : 0;
    const int64_t r = r0 + node;
    const int hq = hk * G + (row_ok ? m - node * G : 0);
    const int lstart = window_of(r);
    const uint32_t* vis = a.mask + r * a.mask_stride;
    asm volatile("prefetch.global.L1 [%0];" ::"l"(vis));
    const float sl2 = fabsf(a.scale) * kTreeLog2e;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    // The additive terms of granules [c0, c1) of this CTA's part, -inf where no slot
    // of the token names the block.  A warp takes 32 slots of one token, or all slots of
    // several; of slots that name one block the lowest counts (in the warp by
    // their lanes, later chunks of a token before earlier ones).
    const int cap = Smem::kCells / nt / NG * NG;
    const int lp = min(pad, 5), span = max(pad, 5);
    int c0 = 0, c1 = 0;
    auto fill = [&](int from) {
      asm volatile("bar.sync 1, 128;" ::: "memory");         // the old terms have been read
      c0 = from;
      c1 = min(from + cap, tiles * NG);
      for (int i = m; i < (c1 - c0) * nt; i += kRows) S.cell[i] = -INFINITY;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      // entry of step j; its bias is loaded a step ahead
      auto entry = [&](int j) {
        return ((warp + (j >> (span - 5) << 2)) << span) + ((~j & ((1 << (span - 5)) - 1)) << 5) + lane;
      };
      auto bias_of = [&](int e) {
        const int slot = e & ((1 << pad) - 1);
        return a.routes.bias && e < entries && slot < K
                   ? __ldg(a.routes.bias + rbase + (int64_t)(e >> pad) * a.routes.row_stride + slot) : 0.0f;
      };
      float next = bias_of(entry(0));
#pragma unroll 1
      for (int j = 0, e = entry(0); e - lane < entries; ++j) {
        const float bias = next;
        const uint32_t v = e >= entries ? 0u : e < Smem::kSlots ? S.slot[e] : remote_of(e);
        const int nd = e >> pad;
        e = entry(j + 1);
        next = bias_of(e);
        // a block's granules follow one another in the union
        const int g = v >> 3;
        int rk = (int)S.before[g >> 5] + __popc(S.bits[g >> 5] & ((1u << (g & 31)) - 1u)) - rank0;
        const int rk1 = min(rk + (int)(v & 7u), c1);
        rk = max(rk, c0);
        const uint32_t same = __match_any_sync(0xffffffffu, v << 5 | (uint32_t)(lane >> lp));
        if (__ffs(same) - 1 == lane) {
          // a finite bias stays finite: its block has keys, if far ones (see kFar)
          const float term = bias >= -FLT_MAX ? fmaxf(bias * kTreeLog2e, -FLT_MAX) : bias;
#pragma unroll 1
          for (float* c = S.cell + (rk - c0) * nt + nd; rk < rk1; ++rk, c += nt) *c = term;
        }
        __syncwarp();
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
    };
    float m_run = -INFINITY, l_run = 0.0f;
    bool alive = true;
#pragma unroll 1
    for (int it = 0; it < tiles; ++it) {
      if (it * NG >= c1) fill(it * NG);
      if (!alive || !warp_on) continue;          // only the table's barriers
      const int sb = it & 1;
      if (!tree_wait_warp(&S.sfull[sb], (uint32_t)(it >> 1) & 1u, abort_flag, derr, 61)) { alive = false; continue; }
      tc_fence_after();
      const uint32_t tS = tmem + sb * kKeys + lane_base;
      float x[kKeys];
      tmem_ld32f(tS, x);
      tmem_ld32f(tS + 32, x + 32);
      // additive term of each granule for this row; pure: one term for all its keys
      float add[NG];
      bool pure = true, none = true, tail = false;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int t0 = S.tok[it & 7][g];
        add[g] = -INFINITY;
        tail |= t0 >= 0 && t0 + GR > end;
        if (t0 >= 0 && row_ok) {
          const bool far = t0 < lstart;
          if (far) add[g] = S.cell[(it * NG + g - c0) * nt + node];
          else if (t0 + GR <= ctx) add[g] = 0.0f;
          const bool p = far ? t0 + GR <= lstart : t0 + GR <= ctx;
          pure &= p;
          none &= p && add[g] == -INFINITY;
        }
      }
      const bool all_none = __all_sync(0xffffffffu, none), all_pure = __all_sync(0xffffffffu, pure);
      if (tail) {
        // V rows behind the last drafted token: P = 0 must not meet a NaN
        const int st = it % kVSlots;
        if (!tree_wait_warp(&S.vfull[st], (uint32_t)(it / kVSlots) & 1u, abort_flag, derr, 60)) alive = false;
        // (16 threads per row of 256 bytes)
#pragma unroll 1
        for (int g = 0; alive && g < NG; ++g) {
          const int t0 = S.tok[it & 7][g];
          uint8_t* v = S.v[st] + ((m & 15) >> 3) * 8192 + g * GR * 128 + ((m & 7) << 4);
          for (int q = t0 < 0 ? GR : max(0, end - t0) + (m >> 4); q < GR; q += nact * 2)
            *reinterpret_cast<uint4*>(v + q * 128) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      if (all_none) {
        // no row of this warp attends the tile
        tmem_ld_wait();
        uint32_t pk[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_st8(tS + c * 8, pk);
      } else {
        float sl = sl2;
        if (!all_pure) {
          // which keys: before the window with the granule's term, window and
          // visible drafted tokens without, nothing else
          uint64_t far = 0, near = 0;
#pragma unroll 1
          for (int g = 0; g < NG; ++g) {
            const int t0 = S.tok[it & 7][g];
            if (t0 < 0 || !row_ok) continue;
            const int rem = min(GR, max(0, lstart - t0)), loc = min(GR, max(0, ctx - t0));
            uint64_t f = rem >= 64 ? ~0ull : (1ull << rem) - 1ull;
            uint64_t on = (loc >= 64 ? ~0ull : (1ull << loc) - 1ull) & ~f;
            if (loc < GR) {
              const int v0 = t0 + loc - ctx;     // drafted token of column loc
              uint64_t bits = 0;
#pragma unroll 1
              for (int w = 0; w < 3; ++w) {
                const int wi = (v0 >> 5) + w, sh = wi * 32 - v0;        // column of the word's first token - loc
                if (wi >= a.mask_words || wi * 32 >= total_n || sh >= 64) break;
                uint32_t mw = __ldg(vis + wi);
                if (total_n - wi * 32 < 32) mw &= (1u << (total_n - wi * 32)) - 1u;
                bits |= sh >= 0 ? (uint64_t)mw << sh : (uint64_t)(mw >> -sh);
              }
              on |= bits << loc;
            }
            if (GR < 64) on &= (1ull << (GR & 63)) - 1ull;
            far |= f << (g * GR & 63);
            near |= on << (g * GR & 63);
          }
          tmem_ld_wait();
          const uint32_t fw[2] = {(uint32_t)far, (uint32_t)(far >> 32)};
          const uint32_t kw[2] = {(uint32_t)(far | near), (uint32_t)((far | near) >> 32)};
#pragma unroll
          for (int c = 0; c < kKeys; ++c) {
            const uint32_t bit = 1u << (c & 31);
            const float y = fmaf(x[c], sl2, fw[c >> 5] & bit ? add[c / GR] : 0.0f);
            x[c] = kw[c >> 5] & bit ? y : -INFINITY;
          }
          sl = 1.0f;                             // x holds logits: nothing is left to add
#pragma unroll
          for (int g = 0; g < NG; ++g) add[g] = 0.0f;
        }
        tmem_ld_wait();
        float mx = -INFINITY;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float h = -INFINITY;
#pragma unroll
          for (int c = 0; c < GR; ++c) h = fmaxf(h, x[g * GR + c]);
          mx = fmaxf(mx, fmaf(h, sl, add[g]));                          // sl >= 0
        }
        // running maximum; O follows it only when it grew by more than 2^kGrow
        const bool grow = mx > m_run + kGrow;
        const bool scale_o = grow && m_run != -INFINITY;
        if (__any_sync(0xffffffffu, scale_o)) {
          const float f = scale_o ? fast_exp2(m_run - mx) : 1.0f;
          if (it > 0) {
            if (!tree_wait_warp(&S.pvdone[(it - 1) & 1], (uint32_t)((it - 1) >> 1) & 1u, abort_flag, derr, 62)) {
              alive = false;
              continue;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 128; c += 16) {
              float o[16];
              tmem_ld16f(tO + c + lane_base, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] *= f;
              tmem_st16f(tO + c + lane_base, o);
            }
            tmem_st_wait();
          }
          l_run *= f;
        }
        if (grow) m_run = mx;
        const float mu = m_run == -INFINITY ? 0.0f : m_run;
        // P is rounded to the caches' type for the matrix product (half a unit
        // in the last place per weight): outputs are off by 0.0023 in bf16 where
        // the rounded output alone gives 0.0017 (relative 2-norms).  A second
        // product with what the rounding leaves would close the gap and was not
        // taken: 82 -> 89 us (32 x 1 token), 47 -> 56 (16 x 16), 33 -> 35 (4 x 64).
        // The sum keeps the unrounded weights because lse is an fp32 result
        uint64_t ls = f2_pack(0.0f, 0.0f);
        const uint64_t slv = f2_pack(sl, sl);
        uint32_t pk[kKeys / 2];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint64_t ad = f2_pack(add[g] - mu, add[g] - mu);
#pragma unroll
          for (int c = 0; c < GR; c += 2) {
            float y0, y1;
            f2_unpack(ffma2(f2_pack(x[g * GR + c], x[g * GR + c + 1]), slv, ad), y0, y1);
            const float p0 = fast_exp2(y0), p1 = fast_exp2(y1);
            ls = fadd2(ls, f2_pack(p0, p1));
            pk[(g * GR + c) >> 1] = pack2(p0, p1, (T*)nullptr);
          }
        }
        tmem_st32(tS, pk);
        float l0, l1;
        f2_unpack(ls, l0, l1);
        l_run += l0 + l1;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.pfull[sb]);
    }
    // ---- the end: O from TMEM ----
    if (warp_on) {
      if (tiles > 0 && alive)
        alive = tree_wait_warp(&S.pvdone[(tiles - 1) & 1], (uint32_t)((tiles - 1) >> 1) & 1u, abort_flag, derr, 63);
      tc_fence_after();
      const float inv = l_run > 0.0f ? 1.0f / l_run : 0.0f;
      T* op = reinterpret_cast<T*>(a.qo.out) + r * a.qo.o_stride_tok + (int64_t)hq * a.qo.o_stride_head;
      float chk = l_run * 0.0f;                  // x * 0 is 0 for a finite x only
#pragma unroll 1
      for (int c = 0; c < 128; c += 32) {
        float o[32];
        tmem_ld32f(tO + c + lane_base, o);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          if (tiles == 0) o[k] = 0.0f;
          chk = fmaf(o[k], 0.0f, chk);
        }
        if (nsp == 1) {
          // the unit is this CTA's alone
          if (row_ok) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              *reinterpret_cast<uint4*>(op + c + v * 8) =
                  make_uint4(pack2(o[8 * v] * inv, o[8 * v + 1] * inv, (T*)nullptr),
                             pack2(o[8 * v + 2] * inv, o[8 * v + 3] * inv, (T*)nullptr),
                             pack2(o[8 * v + 4] * inv, o[8 * v + 5] * inv, (T*)nullptr),
                             pack2(o[8 * v + 6] * inv, o[8 * v + 7] * inv, (T*)nullptr));
          }
        } else {
          // into shared memory (the K and V slots are free)
#pragma unroll
          for (int v = 0; v < 8; ++v)
            *reinterpret_cast<float4*>(S.k[0] + m * 512 + ((((c >> 2) + v) ^ (m & 7)) << 4)) =
                make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
        }
      }
      if (nsp == 1) {
        if (row_ok && a.qo.lse)
          a.qo.lse[r * a.qo.lse_stride_tok + (int64_t)hq * a.qo.lse_stride_head] =
              l_run > 0.0f ? (m_run + log2f(l_run)) * kTreeLn2 : -INFINITY;
        const bool far = m_run < kFar && m_run != -INFINITY;
        redo = __ballot_sync(0xffffffffu, row_ok && (!(chk == 0.0f) || far));
      } else {
        S.m[m] = m_run;
        S.l[m] = tiles > 0 ? l_run : -1.0f;      // -1: this CTA had no tile
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, kTmemCols);
  if (nsp == 1) {
    // (the stores above come before these, and Q is in place for every thread)
    for (; redo; redo &= redo - 1) redo_row<T>(a, sq, s, r0, warp * 32 + __ffs(redo) - 1, G, hk, S.q, QR * 128);
    after_first();
    return;
  }
  cluster.sync();
  // ---- join: row m by CTA m % nsp, a warp per row, lane = 4 dims ----
#pragma unroll 1
  for (int m = split + nsp * warp; m < nrows; m += nsp * (kThreads / 32)) {
    const int node = m / G;
    const int64_t r = r0 + node;
    const int hq = hk * G + m - node * G;
    float mk = -INFINITY, lk = -1.0f;            // lane k holds CTA k's
    if (lane < nsp) {
      mk = *cluster.map_shared_rank(&S.m[m], lane);
      lk = *cluster.map_shared_rank(&S.l[m], lane);
    }
    float M = mk;
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    M = __shfl_sync(0xffffffffu, M, 0);
    // a part without a key for the row has weight 0, and 0 * NaN shows below;
    // one without a tile is left out
    const float wk = mk == -INFINITY ? 0.0f : fast_exp2(mk - M);
    float L = 0.0f;
    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int k0 = 0; k0 < nsp; k0 += 8) {
      float4 o[8];                               // eight parts in flight
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < nsp)
          o[k] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(&S.k[0][0], k0 + k) + m * 512 +
                                                  ((lane ^ (m & 7)) << 4));
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = __shfl_sync(0xffffffffu, wk, k0 + k), l1 = __shfl_sync(0xffffffffu, lk, k0 + k);
        if (l1 != -1.0f) {                       // lanes k >= nsp hold -1
          L += l1 * w;
          O.x += o[k].x * w; O.y += o[k].y * w; O.z += o[k].z * w; O.w += o[k].w * w;
        }
      }
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    const bool fine = (O.x + O.y + O.z + O.w + L) * 0.0f == 0.0f && !(M < kFar && M != -INFINITY);
    if (!__all_sync(0xffffffffu, fine)) {
      redo_row<T>(a, sq, s, r0, m, G, hk, S.q, QR * 128);
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
  after_first();
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

// How the units are cut into CTAs: `whole` units of one CTA each, the rest of `sp` CTAs.
struct TreeCut {
  int64_t whole;
  int sp;
};

// A CTA costs about 10 us before and after its tiles; a tile takes 0.95 us (its chain
// of S, softmax and P V), or what the memory gives: 1.49 us with two CTAs on every SM.
// Past one wave of CTAs the last one is about half full; full waves of whole units with a
// launch of split ones behind them waste less where the units are long.  (Measured,
// us, 1 / 2 / 3 / 8 CTAs per unit: 160 units of 34 tiles 47 / 62 / 53 / 82 (148 whole and
// 12 of 2..6 CTAs 49), 80 of 15 29 / 23 / 21 / 41, 10 of 20 27 / 21 / 19 / 14; 320 of 37
// 100 / 96 / 100 / 152, as 296 whole ones and 24 of 8 CTAs 78; 640 of 24 148 / 157 / 185 /
// 309, as 592 whole ones and 48 of 6 135.)
// More than 8 CTAs, which leave gaps in the GPU's processing clusters, only where most of
// the GPU stays empty otherwise: 10 units of 16 CTAs and 4 units of some 250 tiles (33 ->
// 29 with 16 CTAs) are inside the bound of 160 CTAs, 20 units of 20 tiles (280 CTAs, 17 ->
// 27 with 14) are outside; nothing between the two was measured.
// The number of tiles is not known here.  The union of a tree's routed blocks is taken as
// twice K, which is what the measured trees have (each token K of 2 K blocks); a router
// whose tokens agree more or less shifts the choice, not the result.
static TreeCut tree_cut(const DashTreeAttnArgs& a, int64_t units) {
  if (a.num_splits) return {0, a.num_splits};
  int64_t keys = (int64_t)(a.seqs.max_q_len == 1 ? 1 : 2) * a.routes.K * a.block_size + a.local_window + a.seqs.max_q_len;
  const int64_t most = (int64_t)a.bt_width * a.block_size;
  const double tiles = (double)((keys < most ? keys : most) + kKeys - 1) / kKeys;
  auto best = [&](int64_t n, int& sp) {
    double least = 1e30;
    for (int k = 1; k <= kMaxCluster && k <= tiles && (k <= 8 || n * k <= 160); ++k) {
      const double waves = (double)n * k / 296, tile = waves < 1 ? 1.49 * waves : 1.49;
      const double own = 10.0 + tiles / k * (tile > 0.95 ? tile : 0.95), t = own * (waves <= 1 ? 1.0 : waves + 0.5);
      if (t < least) { least = t; sp = k; }
    }
    return least;
  };
  TreeCut one = {0, 1}, two = {units / 296 * 296, 1};
  const double t1 = best(units, one.sp);
  if (two.whole == 0 || two.whole == units) return one;
  const double t2 = (double)(two.whole / 296) * (10.0 + tiles * 1.49) + best(units - two.whole, two.sp) + 3.0;
  return t2 < t1 ? two : one;
}

template <typename T, int GR, int QR>
static int launch_tc(const DashTreeAttnArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  const int per = kRows / (a.qo.n_heads / a.kv.n_kv_heads);
  const int n_tiles = (a.seqs.max_q_len + per - 1) / per;
  const int64_t units = (int64_t)a.seqs.n_seq * a.kv.n_kv_heads * n_tiles;
  const TreeCut cut = tree_cut(a, units);
  if (units * cut.sp > INT32_MAX) return set_error(DASH_ERR_UNSUPPORTED, "too many sequences x kv heads");
  const int smem = (int)sizeof(TreeSmem<QR>) + 1024;
  auto kernel = tree_tc_kernel<T, GR, QR>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  for (int part = 0; part < 2 && e == cudaSuccess; ++part) {
    const int64_t n = part == 0 ? cut.whole : units - cut.whole;
    if (n == 0) continue;
    const int sp = part == 0 ? 1 : cut.sp;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * sp));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)sp;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = part == 1 && cut.whole > 0 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kernel, mk, mv, a, n_tiles, part == 0 ? 0 : (int)cut.whole,
                           part == 0 && cut.whole < units);
    count_launch();
  }
  if (e != cudaSuccess) return set_error(DASH_ERR_CUDA, "tree_tc_kernel launch failed: %s", cudaGetErrorString(e));
  return check_launch("tree_tc_kernel");
}

template <typename T>
static int launch_tc_gr(const DashTreeAttnArgs& a, cudaStream_t st) {
  const int gr = granule_of(a.block_size);
  CUtensorMap mk, mv;
  int rc = page_map(&mk, a.kv.k, a, gr);
  if (rc == DASH_OK) rc = page_map(&mv, a.kv.v, a, gr);
  if (rc != DASH_OK) return rc;
  const int G = a.qo.n_heads / a.kv.n_kv_heads;
  const int rows = (a.seqs.max_q_len < kRows / G ? a.seqs.max_q_len : kRows / G) * G;
  if (rows <= 32) return gr == 16 ? launch_tc<T, 16, 32>(a, mk, mv, st)
                       : gr == 32 ? launch_tc<T, 32, 32>(a, mk, mv, st) : launch_tc<T, 64, 32>(a, mk, mv, st);
  if (rows <= 64) return gr == 16 ? launch_tc<T, 16, 64>(a, mk, mv, st)
                       : gr == 32 ? launch_tc<T, 32, 64>(a, mk, mv, st) : launch_tc<T, 64, 64>(a, mk, mv, st);
  return gr == 16 ? launch_tc<T, 16, 128>(a, mk, mv, st)
       : gr == 32 ? launch_tc<T, 32, 128>(a, mk, mv, st) : launch_tc<T, 64, 128>(a, mk, mv, st);
}

int launch_tree_tc(const DashTreeAttnArgs& a, cudaStream_t st) {
  return a.kv.dtype == DASH_DTYPE_BF16 ? launch_tc_gr<__nv_bfloat16>(a, st) : launch_tc_gr<__half>(a, st);
}

}  // namespace dash
