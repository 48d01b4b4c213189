// The whole layer for a few tokens (1 <= T <= 64) in one kernel:
//   y[t] = (silu(x Wg^T) * (x Wu^T)) Wd^T + sum_{j<k} g_tj silu(x_t . Up[e_tj]) Down[e_tj]
// with (e, g) the router's product-key selection.  Every weight is used by T tokens only, so the kernel is bound by
// the bytes of Wg, Wu, Wd, the two sub-key matrices and the selected table rows, and by the latencies between its
// dependent parts.
//
// One persistent block per SM, launched cooperatively (its blocks wait on one another).  Every matrix is cut by rows:
// block c owns a contiguous range of gate / up columns, of router sub-keys and of output columns, so all blocks read the
// same number of bytes whatever the sizes.  Inside a block the MLP and the experts go side by side:
//
//   MLP      gate | up rows -> act  --[all act written]-->  down rows  -> + routed sum -> y
//   experts  router rows -> logits  --[all logits written]-->  selection, k dots (a few blocks per token)
//                                   and those k Down rows, a block's share summed --[all partial sums written]-->
//                                   added up for this block's columns
//
// The brackets are counters in global memory; every wait (on them and on barriers in shared memory) is bounded.  Two forms
// of the products (the rule that picks one stands in omni_decode): "direct" streams the weights through registers into
// mma.sync, "ring" by TMA through shared memory into tcgen05.mma.  The expert warps' code is the same in both.
//
// Measured (B200, CUDA graph; floor = bytes at 6547 GB/s): 1 token x 256 x 1024 12.2 us (latency: five dependent passes
// through L2 and a cooperative launch), 1 x 1024 x 4096 15.8 us (floor 3.9), 8 x 4096 x 11008 56.5 us (42.6: 75 % of the
// copy rate), 64 x 2048 x 8192 40.4 us (17.1), 24 x 4096 x 11008 with 64 of 2^20 experts 69.5 us (47.8).
// The layer's four-kernel forward takes 34 us for 1 to 64 tokens of 256 x 1024, where this takes 16 to 23, and 141 us for
// 2048 x 8192, where this takes 34 to 47 (events around one call, cold L2).
//
// act is rounded to bf16 (it is an operand of the down projection); everything else is summed in fp32 and y is rounded
// once.
#include "router_select.cuh"
#include "tcgen05.cuh"

namespace omni {
namespace {

using namespace sel;

using namespace tc;

constexpr int kEpiWarps = 4, kExpWarps = 8;
constexpr int kFirstExp = 2 + kEpiWarps;
constexpr int kDecThreads = 32 * (kFirstExp + kExpWarps);
constexpr int kDecMaxTokens = 64;
constexpr int kSlots = 8;              // at most
constexpr int kSlotBytes = 24 * 1024;  // at least
constexpr int kSmemMost = 226 * 1024;  // dynamic shared memory of a block beside its static part
// counters, one per 128-byte line
enum { CNT_LOGITS = 0, CNT_ACT = 32, CNT_ROUTED = 64, CNT_EXIT = 96, CNT_GROUP = 128, kGroupStride = 8, kMaxGroups = 256,
       CNT_WORDS = CNT_GROUP + kGroupStride * kMaxGroups };
constexpr int kMaxSplit = 4;  // blocks of a group that cuts K

struct DecodeArgs {
  const __nv_bfloat16 *x, *wg, *wu, *wd, *kx, *ky, *up, *down;
  const float *bn_scale, *bn_shift;
  int T, H, I, n, k, kk, cells;
  int64_t N;
  int share;       // blocks that work on one token's dot products
  int rows_r, rows_gu, rows_d;    // weight rows of a box: router, gate (and up), down
  int slot_bytes, slots;          // ring
  int slices_r, slices_gu, slices_d;  // K slices of a slot
  int max_cols;    // output columns of the widest block
  int rsplit, rgroups;            // blocks of a group in the router, number of groups
  int ksplit, groups;             // the same in the down projection
  int m_r, m_gu, m_d;             // M of the tcgen05 tiles: 64 or 128
  int* counters;
  float* logits;   // [rsplit, T, 2n]: partial sums
  float* routed;   // [share, T, H]: partial routed sums
  __nv_bfloat16* act;  // [T, I]
  float* partial;  // [ksplit, T, H]
  __nv_bfloat16* y;
  int32_t* status;
};

constexpr int kScratchBytes = 28 * 1024;  // of the expert warps

// TMEM columns of a block with N tokens: two gate | up accumulators of 2N, down at 4N, router at 5N.
template <int N>
struct DecCfg {
  static constexpr int kTmemCols = 8 * N;
  static constexpr int kDown = 4 * N, kRouter = 5 * N;
};

// The columns and rows of block c.
struct Share {
  int n0, n1;  // router rows that its group works on: x-axis sub-keys, then y-axis ones
  int h0, h1;  // its K slices of them
  int rpart;   // its place in that group
  int c0, c1;  // gate / up columns
  int R0, R1;  // rows of the down projection that its group works on
  int r0, r1;  // ... and those of them that this block writes: its output columns
  int k0, k1;  // its K slices of the down projection
  int part;    // its place in the group
};
// Output columns go in groups of four.
__device__ __forceinline__ Share share_of(const DecodeArgs& a, int c, int G) {
  const auto cut = [](int64_t n, int i, int of) { return static_cast<int>(n * i / of); };
  Share s;
  s.c0 = cut(a.I, c, G), s.c1 = cut(a.I, c + 1, G);
  const int rg = c / a.rsplit, hs = ceil_div(a.H, BK);
  s.rpart = c - rg * a.rsplit;
  s.n0 = rg < a.rgroups ? cut(2 * a.n, rg, a.rgroups) : 0, s.n1 = rg < a.rgroups ? cut(2 * a.n, rg + 1, a.rgroups) : 0;
  s.h0 = cut(hs, s.rpart, a.rsplit), s.h1 = cut(hs, s.rpart + 1, a.rsplit);
  const int grp = c / a.ksplit;
  s.part = c - grp * a.ksplit;
  if (grp >= a.groups) {
    s.R0 = s.R1 = s.r0 = s.r1 = s.k0 = s.k1 = 0;
    return s;
  }
  const int q0 = cut(a.H / 4, grp, a.groups), q1 = cut(a.H / 4, grp + 1, a.groups);
  s.R0 = 4 * q0, s.R1 = 4 * q1;
  s.r0 = 4 * (q0 + cut(q1 - q0, s.part, a.ksplit)), s.r1 = 4 * (q0 + cut(q1 - q0, s.part + 1, a.ksplit));
  const int total = ceil_div(a.I, BK);
  s.k0 = cut(total, s.part, a.ksplit), s.k1 = cut(total, s.part + 1, a.ksplit);
  return s;
}

__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// One thread, after a barrier of the threads whose writes it announces: the release covers them too (barriers are part of
// the causality order).  A fence of its own in front of it would wait for the same writes twice.
__device__ __forceinline__ void signal(int* counter) {
  asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(counter) : "memory");
}
// Bounded: gives up after about two seconds, flags it, and lets the caller go on (its results are then invalid; every
// index that is read afterwards is checked before it is used as an address).
__device__ __forceinline__ void wait_for(const int* counter, int target, int32_t* status) {
#pragma unroll 1
  for (int i = 0; i < (1 << 22); ++i) {
    int v;  // (a relaxed poll and one fence after it: the fence costs 1 us more than the acquiring polls)
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
    if (v >= target) return;
  }
  atomicOr(status, OMNI_ST_WAIT_TIMEOUT);
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// barrier `id` of 256 threads that also says whether any of them has the predicate
__device__ __forceinline__ bool bar_any(int id, int threads, bool pred) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbarrier.cta.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(pred)) : "memory");
  return r != 0;
}
// asks for [p, p + bytes) to come into L2; p and bytes multiples of 16
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 ldg128_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__host__ __device__ __forceinline__ int round8(int v) { return (v + 7) & ~7; }

// ---- MLP --------------------------------------------------------------------------------------
struct Ring {
  uint32_t data, full, empty;  // slots; barriers of 8 bytes each
  volatile int* abort_flag;
};

// One lane.  gate / up tiles of up to 128 columns, then the down rows.
template <int N>
__device__ __forceinline__ void producer(const DecodeArgs& a, const Ring& r, const CUtensorMap* tx, const CUtensorMap* tkx, const CUtensorMap* tky,
                                         const CUtensorMap* tg, const CUtensorMap* tu, const CUtensorMap* td, const CUtensorMap* ta,
                                         const Share& b) {
  int slot = 0;
  uint32_t phase = 1;  // the first pass over the ring finds its slots empty
  const auto next = [&] {
    if (++slot == a.slots) slot = 0, phase ^= 1;
  };
  if (b.n0 < b.n1) {
    // rows [n0, n1) of the two sub-key matrices on top of one another: two boxes at consecutive rows would have to start
    // on a multiple of 8 in shared memory, so a block that has rows of both axes loads them as two halves of the slice
    const int part = round8(a.rows_r) * 128;
    const bool has_x = b.n0 < a.n, has_y = b.n1 > a.n;
    for (int s = b.h0; s < b.h1; s += a.slices_r, next()) {
      if (!mbar_wait(r.empty + 8 * slot, phase, r.abort_flag, a.status)) return;
      const int cnt = min(a.slices_r, b.h1 - s);
      const uint32_t full = r.full + 8 * slot;
      mbar_arrive_expect_tx(full, cnt * ((static_cast<int>(has_x) + static_cast<int>(has_y)) * a.rows_r + N) * 128);
      uint32_t dst = r.data + slot * a.slot_bytes;
      for (int q = 0; q < cnt; ++q, dst += 2 * part + N * 128) {
        if (has_x) tma_load_2d(dst, tkx, (s + q) * BK, b.n0, full);
        if (has_y) tma_load_2d(dst + part, tky, (s + q) * BK, b.n0 < a.n ? 0 : b.n0 - a.n, full);
        tma_load_2d(dst + 2 * part, tx, (s + q) * BK, 0, full);
      }
    }
  }
  {
    const int total = ceil_div(a.H, BK), part = round8(a.rows_gu) * 128;
    for (int col = b.c0; col < b.c1; col += 128) {
      for (int s = 0; s < total; s += a.slices_gu, next()) {
        if (!mbar_wait(r.empty + 8 * slot, phase, r.abort_flag, a.status)) return;
        const int cnt = min(a.slices_gu, total - s);
        const uint32_t full = r.full + 8 * slot;
        mbar_arrive_expect_tx(full, cnt * (2 * a.rows_gu + N) * 128);
        uint32_t dst = r.data + slot * a.slot_bytes;
        for (int q = 0; q < cnt; ++q, dst += 2 * part + N * 128) {
          tma_load_2d(dst, tg, (s + q) * BK, col, full);
          tma_load_2d(dst + part, tu, (s + q) * BK, col, full);
          tma_load_2d(dst + 2 * part, tx, (s + q) * BK, 0, full);
        }
      }
    }
  }
  if (b.R0 == b.R1) return;
  const int part = round8(a.rows_d) * 128;
  const int stages = ceil_div(b.k1 - b.k0, a.slices_d);
  const int ahead = min(a.slots, stages);
  const int slot0 = slot;
  for (int st = 0; st < ahead; ++st, next()) {  // the weights of the first slots do not wait for the activation
    if (!mbar_wait(r.empty + 8 * slot, phase, r.abort_flag, a.status)) return;
    const int s = b.k0 + st * a.slices_d, cnt = min(a.slices_d, b.k1 - s);
    const uint32_t full = r.full + 8 * slot;
    mbar_arrive_expect_tx(full, cnt * (a.rows_d + N) * 128);
    uint32_t dst = r.data + slot * a.slot_bytes;
    for (int q = 0; q < cnt; ++q, dst += part + N * 128) tma_load_2d(dst, td, (s + q) * BK, b.R0, full);
  }
  wait_for(a.counters + CNT_ACT, gridDim.x, a.status);
  asm volatile("fence.proxy.async;" ::: "memory");  // act was written by ordinary stores, the copies below read it
  for (int st = 0, sl = slot0; st < ahead; ++st) {
    const int s = b.k0 + st * a.slices_d, cnt = min(a.slices_d, b.k1 - s);
    uint32_t dst = r.data + sl * a.slot_bytes + part;
    for (int q = 0; q < cnt; ++q, dst += part + N * 128) tma_load_2d(dst, ta, (s + q) * BK, 0, r.full + 8 * sl);
    if (++sl == a.slots) sl = 0;
  }
  for (int st = ahead; st < stages; ++st, next()) {
    if (!mbar_wait(r.empty + 8 * slot, phase, r.abort_flag, a.status)) return;
    const int s = b.k0 + st * a.slices_d, cnt = min(a.slices_d, b.k1 - s);
    const uint32_t full = r.full + 8 * slot;
    mbar_arrive_expect_tx(full, cnt * (a.rows_d + N) * 128);
    uint32_t dst = r.data + slot * a.slot_bytes;
    for (int q = 0; q < cnt; ++q, dst += part + N * 128) {
      tma_load_2d(dst, td, (s + q) * BK, b.R0, full);
      tma_load_2d(dst + part, ta, (s + q) * BK, 0, full);
    }
  }
}

// One lane.  acc_full: one barrier per accumulator (gate | up 0, gate | up 1, down, router); acc_free: of the two gate | up ones.
template <int N>
__device__ __forceinline__ void mma_issuer(const DecodeArgs& a, const Ring& r, uint32_t acc_full, uint32_t acc_free, uint32_t tmem, const Share& b) {
  int slot = 0;
  uint32_t phase = 0;
  const auto next = [&] {
    if (++slot == a.slots) slot = 0, phase ^= 1;
  };
  if (b.n0 < b.n1) {
    const int part = round8(a.rows_r) * 128;
    const uint32_t idesc = make_idesc(a.m_r, N), d = tmem + DecCfg<N>::kRouter;
    for (int s = b.h0; s < b.h1; s += a.slices_r, next()) {
      if (!mbar_wait(r.full + 8 * slot, phase, r.abort_flag, a.status)) return;
      tc_fence_after();
      const int cnt = min(a.slices_r, b.h1 - s);
      uint32_t src = r.data + slot * a.slot_bytes;
      for (int q = 0; q < cnt; ++q, src += 2 * part + N * 128) {
        const uint64_t kd = make_smem_desc(src), bd = make_smem_desc(src + 2 * part);
#pragma unroll
        for (int ks = 0; ks < BK / UMMA_K; ++ks) umma_bf16(d, kd + 2 * ks, bd + 2 * ks, idesc, ((s - b.h0) | q | ks) != 0);
      }
      umma_commit(r.empty + 8 * slot);
    }
    umma_commit(acc_full + 24);
  }
  {
    const int total = ceil_div(a.H, BK), part = round8(a.rows_gu) * 128;
    const uint32_t idesc = make_idesc(a.m_gu, N);
    int it = 0;
    for (int col = b.c0; col < b.c1; col += 128, ++it) {
      const int acc = it & 1;
      if (!mbar_wait(acc_free + 8 * acc, ((it >> 1) & 1) ^ 1, r.abort_flag, a.status)) return;
      tc_fence_after();
      const uint32_t d = tmem + acc * 2 * N;
      for (int s = 0; s < total; s += a.slices_gu, next()) {
        if (!mbar_wait(r.full + 8 * slot, phase, r.abort_flag, a.status)) return;
        tc_fence_after();
        const int cnt = min(a.slices_gu, total - s);
        uint32_t src = r.data + slot * a.slot_bytes;
        for (int q = 0; q < cnt; ++q, src += 2 * part + N * 128) {
          const uint64_t gd = make_smem_desc(src), ud = make_smem_desc(src + part), bd = make_smem_desc(src + 2 * part);
#pragma unroll
          for (int ks = 0; ks < BK / UMMA_K; ++ks) {  // 16 bf16 = 32 bytes = 2 units of the start address
            umma_bf16(d, gd + 2 * ks, bd + 2 * ks, idesc, (s | q | ks) != 0);
            umma_bf16(d + N, ud + 2 * ks, bd + 2 * ks, idesc, (s | q | ks) != 0);
          }
        }
        umma_commit(r.empty + 8 * slot);
      }
      umma_commit(acc_full + 8 * acc);
    }
  }
  if (b.R0 == b.R1) return;
  const int part = round8(a.rows_d) * 128;
  const uint32_t idesc = make_idesc(a.m_d, N);
  const uint32_t d = tmem + DecCfg<N>::kDown;
  for (int s = b.k0; s < b.k1; s += a.slices_d, next()) {
    if (!mbar_wait(r.full + 8 * slot, phase, r.abort_flag, a.status)) return;
    tc_fence_after();
    const int cnt = min(a.slices_d, b.k1 - s);
    uint32_t src = r.data + slot * a.slot_bytes;
    for (int q = 0; q < cnt; ++q, src += part + N * 128) {
      const uint64_t wd = make_smem_desc(src), bd = make_smem_desc(src + part);
#pragma unroll
      for (int ks = 0; ks < BK / UMMA_K; ++ks) umma_bf16(d, wd + 2 * ks, bd + 2 * ks, idesc, ((s - b.k0) | q | ks) != 0);
    }
    umma_commit(r.empty + 8 * slot);
  }
  umma_commit(acc_full + 16);
}

// This block's columns of every token, the partial sums added in block order; all loads of a thread are in flight.  By the
// epilogue and the expert warps together.
constexpr int kFinalThreads = 32 * (kEpiWarps + kExpWarps);
__device__ __forceinline__ void final_sums(const DecodeArgs& a, const float* routed, const Share& b, int tid) {
  const int cols = b.r1 - b.r0;
#pragma unroll 1
  for (int e0 = tid; e0 < a.T * cols; e0 += 4 * kFinalThreads) {
    float v[4][kMaxSplit];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int e = e0 + q * kFinalThreads, t = e / cols, col = e - t * cols;
#pragma unroll
      for (int p = 0; p < kMaxSplit; ++p)
        v[q][p] = p < a.ksplit && t < a.T ? __ldcg(a.partial + (static_cast<int64_t>(p) * a.T + t) * a.H + b.r0 + col) : 0.f;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int e = e0 + q * kFinalThreads, t = e / cols, col = e - t * cols;
      float sum = 0.f;
#pragma unroll
      for (int p = 0; p < kMaxSplit; ++p) sum += v[q][p];
      if (t < a.T) a.y[static_cast<int64_t>(t) * a.H + b.r0 + col] = __float2bfloat16_rn(sum + routed[t * a.max_cols + col]);
    }
  }
}

// The rows of an M = 128 tile lie in TMEM lanes 0 .. 127, those of an M = 64 tile in the first 16 lanes of each quarter
// (a warp may read the quarter that its id selects).  16 tokens at a time.
template <int N>
__device__ __forceinline__ void epilogue(const DecodeArgs& a, const Ring& r, uint32_t acc_full, uint32_t acc_free, uint32_t tmem, const float* routed,
                                         const Share& b) {
  const int warp = threadIdx.x >> 5, lane = lane_id();
  const int quarter = warp & 3;
  const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
  const auto row_of = [&](int m) { return m == 128 ? quarter * 32 + lane : (lane < 16 ? quarter * 16 + lane : 1 << 20); };
  const auto first_row = [&](int m) { return m == 128 ? quarter * 32 : quarter * 16; };
  if (b.n0 < b.n1) {
    // tile row i < round8(rows_r) is the i-th x-axis row of the group, the rows after that the y-axis ones
    const bool ok = __all_sync(FULL_MASK, mbar_wait(acc_full + 24, 0, r.abort_flag, a.status));
    tc_fence_after();
    const int row = row_of(a.m_r), half = round8(a.rows_r), nx = b.n0 < a.n ? min(b.n1, a.n) - b.n0 : 0;
    const int key = row < half ? (row < nx ? b.n0 + row : -1) : (b.n0 + nx + row - half < b.n1 ? b.n0 + nx + row - half : -1);
    if (ok && first_row(a.m_r) < 2 * half) {
#pragma unroll 1
      for (int t0 = 0; t0 < a.T; t0 += 16) {
        uint32_t ra[16];
        tmem_ld16(tmem + lanes + DecCfg<N>::kRouter + t0, ra);
        if (key >= 0) {
          float* out = a.logits + (static_cast<int64_t>(b.rpart) * a.T + t0) * (2 * a.n) + key;
#pragma unroll
          for (int t = 0; t < 16; ++t)
            if (t0 + t < a.T) __stcg(out + static_cast<int64_t>(t) * (2 * a.n), __uint_as_float(ra[t]));
        }
      }
    }
  }
  bar_sync(1, 32 * kEpiWarps);
  if (threadIdx.x == 64) signal(a.counters + CNT_LOGITS);
  int it = 0;
  for (int col = b.c0; col < b.c1; col += 128, ++it) {
    const int acc = it & 1, rows = min(128, b.c1 - col), row = row_of(a.m_gu);
    const bool ok = __all_sync(FULL_MASK, mbar_wait(acc_full + 8 * acc, (it >> 1) & 1, r.abort_flag, a.status));
    tc_fence_after();
    if (ok && first_row(a.m_gu) < rows) {
      const uint32_t d = tmem + lanes + acc * 2 * N;
#pragma unroll 1
      for (int t0 = 0; t0 < a.T; t0 += 16) {  // (rolled: code that runs once is paid for in instruction fetches)
        uint32_t ra[16], rb[16];
        tmem_ld16(d + t0, ra);
        tmem_ld16(d + N + t0, rb);
        if (row < rows) {
          __nv_bfloat16* out = a.act + static_cast<int64_t>(t0) * a.I + col + row;
          __nv_bfloat16 v[16];
#pragma unroll
          for (int t = 0; t < 16; ++t) v[t] = __float2bfloat16_rn(silu_fast(__uint_as_float(ra[t])) * __uint_as_float(rb[t]));
#pragma unroll
          for (int t = 0; t < 16; ++t)
            if (t0 + t < a.T) out[static_cast<int64_t>(t) * a.I] = v[t];
        }
      }
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(acc_free + 8 * acc);
  }
  asm volatile("fence.proxy.async;" ::: "memory");
  bar_sync(1, 32 * kEpiWarps);
  if (threadIdx.x == 64) signal(a.counters + CNT_ACT);
  if (b.R0 == b.R1) {
    bar_sync(3, kFinalThreads);
    return;
  }
  const int row = row_of(a.m_d), rows = b.R1 - b.R0;
  const bool ok = __all_sync(FULL_MASK, mbar_wait(acc_full + 16, 0, r.abort_flag, a.status));
  tc_fence_after();
  if (ok && first_row(a.m_d) < rows) {
#pragma unroll 1
    for (int t0 = 0; t0 < a.T; t0 += 16) {
      uint32_t ra[16];
      tmem_ld16(tmem + lanes + DecCfg<N>::kDown + t0, ra);
      if (row < rows) {
        float* out = a.partial + (static_cast<int64_t>(b.part) * a.T + t0) * a.H + b.R0 + row;
#pragma unroll
        for (int t = 0; t < 16; ++t)
          if (t0 + t < a.T) __stcg(out + static_cast<int64_t>(t) * a.H, __uint_as_float(ra[t]));
      }
    }
  }
  bar_sync(1, 32 * kEpiWarps);
  if (threadIdx.x == 64 && a.ksplit > 1) {
    int* counter = a.counters + CNT_GROUP + kGroupStride * (blockIdx.x / a.ksplit);
    signal(counter);
    wait_for(counter, a.ksplit, a.status);
  }
  bar_sync(3, kFinalThreads);  // the group's partial sums are written, the routed sums are in shared memory
  final_sums(a, routed, b, threadIdx.x - 64);
  tc_fence_before();
}

// ---- expert warps -----------------------------------------------------------------------------
constexpr int kExpThreads = 32 * kExpWarps;
static_assert(kExpThreads == 256, "the selection gives half of the expert threads to each axis");

struct __align__(16) ExpertShared {
  uint32_t top[2][128];        // per axis: every thread's largest key
  float2 red[2][4];
  float val[2][kMaxK];         // the best sub-keys of each axis: log-probability and index
  int idx[2][kMaxK];
  float weight[kMaxK];         // the selection
  int index[kMaxK];
  uint16_t cell[kMaxCells + 8];  // the cells (i, j) of the pruned search, i | j << 8
  int scan[4];
  int count[2], cells;
  uint32_t tau[2], last;
};
// In the scratch, while a token is selected.
struct __align__(16) SelectScratch {
  uint32_t key[2][1024];       // all keys of an axis (for the exact search)
  uint32_t cand[2][1024 + 4];  // keys that can be among the best, and where they stand
  uint16_t cand_at[2][1024];
  uint32_t cell_key[kMaxCells + 4], cell_flat[kMaxCells];
};
static_assert(sizeof(SelectScratch) <= kScratchBytes, "scratch of the expert warps");

// The rank of (mine, id) among the keys all[0 .. n) (descending): how many others are at least `mine`; entries from n to
// the next multiple of 4 are readable and 0.  With `ties`, equal keys are ranked by their ids (ascending), which is a
// second look that only tokens with equal keys pay for.
template <typename Id>
__device__ __forceinline__ int rank_of(const uint32_t* all, int n, uint32_t mine, bool ties, const Id* ids, uint32_t id) {
  const uint4* p = reinterpret_cast<const uint4*>(all);
  int r = -1;
#pragma unroll 4
  for (int q = 0; q < (n + 3) >> 2; ++q) {
    const uint4 o = p[q];
    r += (o.x >= mine) + (o.y >= mine) + (o.z >= mine) + (o.w >= mine);
  }
  if (ties) {
#pragma unroll 1
    for (int q = 0; q < n; ++q) r -= all[q] == mine && (ids ? static_cast<uint32_t>(ids[q]) : static_cast<uint32_t>(q)) > id;
  }
  return r;
}

// Cells (i+1)(j+1) <= k of the kk x kk grid in rank space, row by row (see router_select.cuh).  Returns the number of cells
// in row tid (kk where there is no such row).
__device__ __forceinline__ int fill_cells(ExpertShared& sh, int kk, int k, int tid) {
  const int lane = tid & 31;
  const int mine = tid < kk ? min(kk, k / (tid + 1)) : 0;  // kk <= 128: the first four warps
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(FULL_MASK, sum, o);
    if (lane >= o) sum += v;
  }
  if (tid < 128 && lane == 31) sh.scan[tid >> 5] = sum;
  bar_sync(2, kExpThreads);
  if (tid < kk) {
    int at = sum - mine;
    for (int w = 0; w < (tid >> 5); ++w) at += sh.scan[w];
#pragma unroll 1
    for (int j = 0; j < mine; ++j) sh.cell[at + j] = static_cast<uint16_t>(tid | (j << 8));
  }
  return tid < kk ? mine : kk;
}

// The same result from all kk x kk cells, by one warp: round after round the best entry that comes after the previous
// one in the order (key descending, index ascending), first on each axis, then over the cells.  For the rare token whose
// last score is tied with a cell outside the pruned region.
__device__ __noinline__ void select_exactly(int n, int k, int kk, ExpertShared& sh, const SelectScratch& w) {
  const int lane = lane_id();
  for (int job = 0; job < 3; ++job) {
    const int count = job < 2 ? n : kk * kk, rounds = job < 2 ? kk : k;
    uint32_t pk = 0xffffffffu, pf = 0;
    for (int r = 0; r < rounds; ++r) {
      uint32_t bk = 0, bf = 0xffffffffu;
      for (int q = lane; q < count; q += 32) {
        uint32_t kq, flat;
        if (job < 2) {
          kq = w.key[job][q], flat = q;
        } else {
          const int x = q / kk, y = q - x * kk;
          kq = float_to_key(__fadd_rn(sh.val[0][x], sh.val[1][y]));
          flat = static_cast<uint32_t>(sh.idx[0][x]) * n + sh.idx[1][y];
        }
        const bool after = r == 0 || kq < pk || (kq == pk && flat > pf);
        if (after && (kq > bk || (kq == bk && flat < bf))) bk = kq, bf = flat;
      }
      pk = __reduce_max_sync(FULL_MASK, bk);
      pf = __reduce_min_sync(FULL_MASK, bk == pk ? bf : 0xffffffffu);
      if (lane == 0) {
        if (job < 2) sh.val[job][r] = key_to_float(pk), sh.idx[job][r] = static_cast<int>(pf);
        else sh.weight[r] = expf(key_to_float(pk)), sh.index[r] = static_cast<int>(pf);
      }
    }
    __syncwarp();
  }
}

// The routing of one token, by 256 threads: the first 128 have the x axis, the others the y axis, up to 8 logits each.
// Same definition as select_token in router_select.cuh (scores descending, lower expert index on ties), organised for
// the latency of one token instead of the throughput of many: an entry's rank is the number of keys that are at least
// its own, which has no dependency chain.  With more than 128 entries an axis is thinned first: the kk-th largest of the
// 128 threads' maxima is a lower bound of the kk-th largest entry, and few more entries reach it.  Leaves the selection
// in sh.index / sh.weight, ending with a barrier.
// j0: column of the first cell outside the pruned region in row tid, kk or more where there is none.
__device__ __forceinline__ void select_by_block(const DecodeArgs& a, int t, ExpertShared& sh, SelectScratch& w, int tid, int j0) {
  const int axis = tid >> 7, i = tid & 127, lane = tid & 31, quad = (tid >> 5) & 3;
  const int n = a.n, k = a.k, kk = a.kk;
  const int64_t plane = static_cast<int64_t>(a.T) * (2 * n);
  const float* z = a.logits + static_cast<int64_t>(t) * (2 * n) + axis * n;
  // a thread has the entries i, i + 128, ...: up to 8
  const int per = (n + 127) >> 7;
  // every load is issued before any value is used: no branch stands between them
  float v[8];
  float mx = -INFINITY;
  {
    float q[8][kMaxSplit], sc[8], sf[8];
    const bool bn = a.bn_scale != nullptr;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = e * 128 + i;
      const bool in = c < n;
#pragma unroll
      for (int p = 0; p < kMaxSplit; ++p) q[e][p] = in && p < a.rsplit ? __ldcg(z + p * plane + c) : 0.f;
      sc[e] = in && bn ? __ldg(a.bn_scale + axis * n + c) : 1.f;
      sf[e] = in && bn ? __ldg(a.bn_shift + axis * n + c) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float sum = (q[e][0] + q[e][1]) + (q[e][2] + q[e][3]);
      v[e] = e * 128 + i < n ? (bn ? __fmaf_rn(sum, sc[e], sf[e]) : sum) : -INFINITY;
      mx = fmaxf(mx, v[e]);
    }
  }
  if (i == 0) sh.count[axis] = 0, sh.tau[axis] = 0xffffffffu;
  if (i < kk) sh.idx[axis][i] = -1;
  if (tid < k) sh.index[tid] = -1;
  // maximum and sum of a warp relative to its own maximum, then of the four warps
  mx = warp_max(mx);
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < per) sum += v[e] == -INFINITY ? 0.f : __expf(v[e] - mx);
  sum = warp_sum(sum);
  if (lane == 0) sh.red[axis][quad] = make_float2(mx, sum);
  bar_sync(2, kExpThreads);
  float all_max = sh.red[axis][0].x, all_sum = 0.f;
#pragma unroll
  for (int q = 1; q < 4; ++q) all_max = fmaxf(all_max, sh.red[axis][q].x);
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (sh.red[axis][q].x != -INFINITY) all_sum += sh.red[axis][q].y * __expf(sh.red[axis][q].x - all_max);
  const float lse = logf(all_sum);
  uint32_t key[8];
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    key[e] = 0;
    if (e < per && e * 128 + i < n) {
      key[e] = float_to_key((v[e] - all_max) - lse);
      w.key[axis][e * 128 + i] = key[e];
      top = max(top, key[e]);
    }
  }
  sh.top[axis][i] = top;
  bar_sync(2, kExpThreads);
  // The first round takes all keys for distinct.  Equal ones leave a rank without an entry, which the second round ranks
  // by index.
#pragma unroll 1
  for (int round = 0; round < 2; ++round) {
    const bool ties = round > 0;
    const int width = min(n, 128);
    if (n <= 128) {
      if (i < n) {
        const int r = rank_of<uint16_t>(sh.top[axis], width, top, ties, nullptr, i);
        if (r < kk) sh.val[axis][r] = key_to_float(top), sh.idx[axis][r] = i;
      }
    } else {
      if (i == 0) sh.count[axis] = 0;
      if (rank_of<uint16_t>(sh.top[axis], width, top, ties, nullptr, i) == kk - 1) sh.tau[axis] = top;
      bar_sync(2, kExpThreads);
      const uint32_t tau = sh.tau[axis];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e * 128 + i < n && key[e] >= tau) {
          const int at = atomicAdd(&sh.count[axis], 1);
          w.cand[axis][at] = key[e], w.cand_at[axis][at] = static_cast<uint16_t>(e * 128 + i);
        }
      }
      bar_sync(2, kExpThreads);
      const int m = sh.count[axis];
      if (i < 3 && m + i < ((m + 3) & ~3)) w.cand[axis][m + i] = 0;
      bar_sync(2, kExpThreads);
#pragma unroll 1
      for (int q = i; q < m; q += 128) {
        const uint32_t mine = w.cand[axis][q], at = w.cand_at[axis][q];
        const int r = rank_of(w.cand[axis], m, mine, ties, w.cand_at[axis], at);
        if (r < kk) sh.val[axis][r] = key_to_float(mine), sh.idx[axis][r] = static_cast<int>(at);
      }
    }
    int cells = a.cells;
    if (a.cells <= 128) {
      bar_sync(2, kExpThreads);
      if (tid < ((a.cells + 3) & ~3)) {
        uint32_t kq = 0;
        if (tid < a.cells) {
          const int cell = sh.cell[tid], x = cell & 0xff, y = cell >> 8;
          kq = float_to_key(__fadd_rn(sh.val[0][x], sh.val[1][y]));
          w.cell_flat[tid] = static_cast<uint32_t>(sh.idx[0][x]) * n + sh.idx[1][y];
        }
        w.cell_key[tid] = kq;
      }
    } else {
      // Many cells are thinned too.  The x best of one axis and the ceil(k / x) best of the other make k cells, none below
      // that of the two last ranks, whatever x is: a lower bound of the last score.  (280 cells, k = 64: ranking 4.1 ->
      // 1.5 us, thinning 2 us less than the rest of that; at 50 cells it would cost 1 us and save nothing.)
      if (tid == 0) sh.cells = 0;
      bar_sync(2, kExpThreads);
      uint32_t least = 0;
#pragma unroll 1
      for (int x = 1; x <= kk; x *= 2) {
        const int y = (k + x - 1) / x;
        if (y <= kk) least = max(least, float_to_key(__fadd_rn(sh.val[0][x - 1], sh.val[1][y - 1])));
      }
#pragma unroll 1
      for (int q = tid; q < a.cells; q += kExpThreads) {
        const int cell = sh.cell[q], x = cell & 0xff, y = cell >> 8;
        const uint32_t kq = float_to_key(__fadd_rn(sh.val[0][x], sh.val[1][y]));
        if (kq >= least) {
          const int at = atomicAdd(&sh.cells, 1);
          w.cell_key[at] = kq, w.cell_flat[at] = static_cast<uint32_t>(sh.idx[0][x]) * n + sh.idx[1][y];
        }
      }
      bar_sync(2, kExpThreads);
      cells = sh.cells;
      if (tid < 3 && cells + tid < ((cells + 3) & ~3)) w.cell_key[cells + tid] = 0;
    }
    bar_sync(2, kExpThreads);
#pragma unroll 1
    for (int q = tid; q < cells; q += kExpThreads) {
      const uint32_t mine = w.cell_key[q], flat = w.cell_flat[q];
      const int r = rank_of(w.cell_key, cells, mine, ties, w.cell_flat, flat);
      if (r < k) {
        sh.index[r] = static_cast<int>(flat), sh.weight[r] = expf(key_to_float(mine));
        if (r == k - 1) sh.last = mine;
      }
    }
    bar_sync(2, kExpThreads);
    const bool missing = (i < kk && sh.idx[axis][i] < 0) || (tid < k && sh.index[tid] < 0);
    // a cell outside the pruned region that ties with the last score
    const bool odd = j0 < kk && float_to_key(__fadd_rn(sh.val[0][tid], sh.val[1][j0])) >= sh.last;
    if (!bar_any(2, kExpThreads, missing || odd)) return;
    if (!bar_any(2, kExpThreads, missing)) break;
  }
  if (tid < 32) select_exactly(n, k, kk, sh, w);
  bar_sync(2, kExpThreads);
}

// first_warp: the first of the kExpWarps warps that call this.  The code is kept small: it runs once a launch, and what
// unrolling saves in latency it costs in instruction fetches (two rows of a dot product in flight instead of one: slower).
__device__ __forceinline__ void expert_path(const DecodeArgs& a, ExpertShared& sh, uint8_t* scratch, float* routed, const Share& b, int first_warp) {
  const int warp = (threadIdx.x >> 5) - first_warp, lane = lane_id();
  const int tid = threadIdx.x - 32 * first_warp;
  const int T = a.T, H8 = a.H / 8, k = a.k;
  const int G = gridDim.x, c = blockIdx.x;
  // selection and dot products: `share` blocks per token, each selects (the same routing) and takes every share-th rank
  const int tasks = T * a.share;
  if (c < tasks) {
    const int j0 = fill_cells(sh, a.kk, k, tid);
    if (tid == 0) wait_for(a.counters + CNT_LOGITS, G, a.status);
    bar_sync(2, kExpThreads);
    for (int task = c; task < tasks; task += G) {
      const int t = task / a.share, part_id = task - t * a.share;
      select_by_block(a, t, sh, *reinterpret_cast<SelectScratch*>(scratch), tid, j0);
      // the Down rows of this block's ranks are asked into L2 now, for the sums after the dots
      {
        const int j = part_id + a.share * tid;
        if (j < k && sh.index[j] >= 0 && sh.index[j] < a.N) prefetch_l2(a.down + static_cast<int64_t>(sh.index[j]) * a.H, 2 * a.H);
      }
      const uint4* xr = reinterpret_cast<const uint4*>(a.x + static_cast<int64_t>(t) * a.H);
      for (int j = part_id + a.share * warp; j < k; j += a.share * kExpWarps) {
        const int e = sh.index[j];
        float dot = 0.f;
        const bool ok = e >= 0 && e < a.N;
        if (ok) {
          const uint4* ur = reinterpret_cast<const uint4*>(a.up + static_cast<int64_t>(e) * a.H);
#pragma unroll 1
          for (int p0 = lane; p0 < H8; p0 += 32 * 8) {
            uint4 u[8], v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int p = p0 + 32 * q;
              u[q] = p < H8 ? ldg128_stream(ur + p) : make_uint4(0, 0, 0, 0);
              v[q] = p < H8 ? __ldg(xr + p) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const uint32_t uw[4] = {u[q].x, u[q].y, u[q].z, u[q].w}, vw[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
              for (int d = 0; d < 4; ++d) {
                const float2 uf = bf16x2_to_float2(uw[d]), vf = bf16x2_to_float2(vw[d]);
                dot = __fmaf_rn(uf.x, vf.x, dot), dot = __fmaf_rn(uf.y, vf.y, dot);
              }
            }
          }
        }
        dot = warp_sum(dot);
        if (lane == 0) {
          if (!ok) atomicOr(a.status, OMNI_ST_BAD_EXPERT_INDEX);
          sh.weight[j] = ok ? sh.weight[j] * silu(dot) : 0.f;
          if (!ok) sh.index[j] = 0;
        }
      }
      bar_sync(2, kExpThreads);
      // this share of the token's routed sum, 8 neighbouring columns a thread, 8 rows in flight.  (Whole rows in the block
      // that has their coefficients: when every block read its own columns of the rows of all tokens, each row's page went
      // through every multiprocessor: 17 us after the last coefficient at 24 tokens x 64 rows of 4096, so 4.)
      const int mine = (k - part_id + a.share - 1) / a.share;
      float* out = a.routed + (static_cast<int64_t>(part_id) * T + t) * a.H;
#pragma unroll 1
      for (int p = tid; p < H8; p += kExpThreads) {
        float s[8] = {};
#pragma unroll 1
        for (int m = 0; m < mine; m += 8) {
          uint4 d[8];
          float cf[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int j = part_id + a.share * (m + q);
            const bool in = m + q < mine;
            cf[q] = in ? sh.weight[j] : 0.f;
            d[q] = in ? ldg128_stream(a.down + static_cast<int64_t>(sh.index[j]) * a.H + 8 * p) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const uint32_t dw[4] = {d[q].x, d[q].y, d[q].z, d[q].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = bf16x2_to_float2(dw[i]);
              s[2 * i] = __fmaf_rn(cf[q], f.x, s[2 * i]), s[2 * i + 1] = __fmaf_rn(cf[q], f.y, s[2 * i + 1]);
            }
          }
        }
        __stcg(reinterpret_cast<float4*>(out + 8 * p), make_float4(s[0], s[1], s[2], s[3]));
        __stcg(reinterpret_cast<float4*>(out + 8 * p) + 1, make_float4(s[4], s[5], s[6], s[7]));
      }
      bar_sync(2, kExpThreads);
      if (tid == 0) signal(a.counters + CNT_ROUTED);
    }
  }
  // this block's output columns of every token, the shares added in order
  if (tid == 0) wait_for(a.counters + CNT_ROUTED, tasks, a.status);
  bar_sync(2, kExpThreads);
  const int cols = b.r1 - b.r0;
  const int64_t plane = static_cast<int64_t>(T) * a.H;
#pragma unroll 1
  for (int e = tid; e < T * cols; e += kExpThreads) {
    const int t = e / cols, col = e - t * cols;
    const float* p = a.routed + static_cast<int64_t>(t) * a.H + b.r0 + col;
    float sum = 0.f;
#pragma unroll 1
    for (int q0 = 0; q0 < a.share; q0 += 8) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = q0 + q < a.share ? __ldcg(p + (q0 + q) * plane) : 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) sum += v[q];
    }
    routed[t * a.max_cols + col] = sum;
  }
}

// One thread of a block that has nothing left to do: the last block out leaves the counters as it found them, zero, for
// the next launch on this workspace.
__device__ __forceinline__ void leave(const DecodeArgs& a) {
  if (threadIdx.x != 0) return;
  __threadfence();
  if (atomicAdd(a.counters + CNT_EXIT, 1) == static_cast<int>(gridDim.x) - 1) {
    a.counters[CNT_LOGITS] = 0, a.counters[CNT_ACT] = 0, a.counters[CNT_ROUTED] = 0, a.counters[CNT_EXIT] = 0;
    if (a.ksplit > 1)
      for (int i = 0; i < a.groups; ++i) a.counters[CNT_GROUP + kGroupStride * i] = 0;
    __threadfence();
  }
}

// ---- the direct form --------------------------------------------------------------------------
// For few tokens and few bytes a block the latencies of the ring (descriptor, copy, barrier, TMEM) and of the partial
// sums' exchange weigh more than what they save.  Here eight warps bring the weight rows straight into registers, as the
// A operand (16 rows) of mma.sync.m16n8k16 with 8 tokens as the B operand.  The contraction index may be permuted as long
// as both operands agree: lane (g, t) loads 16 contiguous bytes of row g (four lanes cover 64 bytes = two whole sectors)
// and uses its four words as fragments of two MMAs; the B words are the same 16 bytes of token g's row.  No staging, no
// shuffles; the warps cut K between them and add their sums through shared memory in a fixed order.
constexpr int kMainWarps = 8;
constexpr int kDirThreads = 32 * (kMainWarps + kExpWarps);

// By token tiles of 8 (NT): TG weight tiles share the B fragments, D steps of 32 along K (256 bytes of a row) are loaded
// before the first is used, CAP tiles are summed over the warps at a time.
template <int NT>
struct DirectCfg {
  static constexpr int TG = 2;
  static constexpr int D = 4;
  static constexpr int CAP = NT == 1 ? 12 : 8;
  static constexpr int kPartBytes = kMainWarps * CAP * NT * 128 * 4;
};
static_assert(kExpWarps * 2 * 128 * 4 <= kScratchBytes, "scratch of the expert warps");

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// acc[tile] += (16 weight rows) x (8 NT tokens) over the 32-wide steps [s0, s1) of K = 8 * K8.  row[tile][half]: this
// lane's weight row g (half 0) or g + 8 (half 1), or null.  COHERENT: B was written in this launch.
template <int NT, int TG, int D, bool COHERENT>
__device__ __forceinline__ void mma_rows(float (&acc)[TG][NT][4], const __nv_bfloat16* const (&row)[TG][2], const __nv_bfloat16* B,
                                         int T, int K8, int s0, int s1) {
  const int lane = lane_id(), g = lane >> 2, t = lane & 3;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int s = s0; s < s1; s += D) {
    uint4 a[D][TG][2], b[D][NT];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int piece = (s + d) * 4 + t;
      const bool in = s + d < s1 && piece < K8;
#pragma unroll
      for (int q = 0; q < TG; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) a[d][q][h] = in && row[q][h] ? ldg128_stream(row[q][h] + 8 * piece) : zero;
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int piece = (s + d) * 4 + t;
      const bool in = s + d < s1 && piece < K8;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int tok = nt * 8 + g;
        const __nv_bfloat16* p = B + (static_cast<int64_t>(tok) * K8 + piece) * 8;
        b[d][nt] = in && tok < T ? (COHERENT ? __ldcg(reinterpret_cast<const uint4*>(p)) : ldg128(p)) : zero;
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
      for (int q = 0; q < TG; ++q)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_16816(acc[q][nt], a[d][q][0].x, a[d][q][1].x, a[d][q][0].y, a[d][q][1].y, b[d][nt].x, b[d][nt].y);
          mma_16816(acc[q][nt], a[d][q][0].z, a[d][q][1].z, a[d][q][0].w, a[d][q][1].w, b[d][nt].z, b[d][nt].w);
        }
  }
}

// Accumulators of one tile into part[nt][row][token].
template <int NT>
__device__ __forceinline__ void put_tile(float* part, const float (&acc)[NT][4]) {
  const int lane = lane_id(), g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    *reinterpret_cast<float2*>(part + nt * 128 + g * 8 + 2 * t) = make_float2(acc[nt][0], acc[nt][1]);
    *reinterpret_cast<float2*>(part + nt * 128 + (g + 8) * 8 + 2 * t) = make_float2(acc[nt][2], acc[nt][3]);
  }
}

template <int NT>
__device__ __forceinline__ void main_path(const DecodeArgs& a, float* part, const float* routed, const Share& b) {
  using C = DirectCfg<NT>;
  const int c0 = b.c0, c1 = b.c1, r0 = b.r0, r1 = b.r1;
  const int warp = threadIdx.x >> 5, g = lane_id() >> 2;
  const int tid = threadIdx.x;  // main warps come first
  constexpr int kThr = 32 * kMainWarps;
  const int T = a.T;
  // gate | up: a tile is 8 columns, its A rows 0..7 the gate rows, 8..15 the up rows
  {
    const int K8 = a.H / 8, S = ceil_div(a.H, 32);
    const int s0 = S * warp / kMainWarps, s1 = S * (warp + 1) / kMainWarps;
    const int tiles = ceil_div(c1 - c0, 8);
    for (int base = 0; base < tiles; base += C::CAP) {
      const int cnt = min(C::CAP, tiles - base);
      for (int q0 = 0; q0 < cnt; q0 += C::TG) {
        const __nv_bfloat16* row[C::TG][2];
        float acc[C::TG][NT][4] = {};
#pragma unroll
        for (int q = 0; q < C::TG; ++q) {
          const int col = c0 + (base + q0 + q) * 8 + g;
          const bool ok = q0 + q < cnt && col < c1;
          row[q][0] = ok ? a.wg + static_cast<int64_t>(col) * a.H : nullptr;
          row[q][1] = ok ? a.wu + static_cast<int64_t>(col) * a.H : nullptr;
        }
        mma_rows<NT, C::TG, C::D, false>(acc, row, a.x, T, K8, s0, s1);
#pragma unroll
        for (int q = 0; q < C::TG; ++q)
          if (q0 + q < cnt) put_tile<NT>(part + ((warp * C::CAP + q0 + q) * NT) * 128, acc[q]);
      }
      bar_sync(1, kThr);
      for (int e = tid; e < cnt * NT * 64; e += kThr) {
        const int tok8 = e & 7, col8 = (e >> 3) & 7, nt = (e >> 6) % NT, tile = (e >> 6) / NT;
        const int tok = nt * 8 + tok8, col = c0 + (base + tile) * 8 + col8;
        if (tok < T && col < c1) {
          float gv = 0.f, uv = 0.f;
#pragma unroll
          for (int w = 0; w < kMainWarps; ++w) {
            const float* p = part + ((w * C::CAP + tile) * NT + nt) * 128 + col8 * 8 + tok8;
            gv += p[0], uv += p[64];
          }
          a.act[static_cast<int64_t>(tok) * a.I + col] = __float2bfloat16_rn(silu_fast(gv) * uv);
        }
      }
      bar_sync(1, kThr);
    }
  }
  if (tid == 0) {
    signal(a.counters + CNT_ACT);
    wait_for(a.counters + CNT_ACT, gridDim.x, a.status);
  }
  bar_sync(1, kThr);
  // down: a tile is 16 output columns
  {
    const int K8 = a.I / 8, S = ceil_div(a.I, 32);
    const int s0 = S * warp / kMainWarps, s1 = S * (warp + 1) / kMainWarps;
    const int tiles = ceil_div(r1 - r0, 16);
    bool first = true;
    for (int base = 0; base < tiles; base += C::CAP) {
      const int cnt = min(C::CAP, tiles - base);
      for (int q0 = 0; q0 < cnt; q0 += C::TG) {
        const __nv_bfloat16* row[C::TG][2];
        float acc[C::TG][NT][4] = {};
#pragma unroll
        for (int q = 0; q < C::TG; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = r0 + (base + q0 + q) * 16 + 8 * h + g;
            row[q][h] = q0 + q < cnt && r < r1 ? a.wd + static_cast<int64_t>(r) * a.I : nullptr;
          }
        mma_rows<NT, C::TG, C::D, true>(acc, row, a.act, T, K8, s0, s1);
#pragma unroll
        for (int q = 0; q < C::TG; ++q)
          if (q0 + q < cnt) put_tile<NT>(part + ((warp * C::CAP + q0 + q) * NT) * 128, acc[q]);
      }
      if (first) bar_sync(3, kDirThreads);  // the expert warps have left the routed sums in shared memory
      else bar_sync(1, kThr);
      first = false;
      for (int e = tid; e < cnt * NT * 128; e += kThr) {
        const int row16 = e & 15, tok8 = (e >> 4) & 7, nt = (e >> 7) % NT, tile = (e >> 7) / NT;
        const int tok = nt * 8 + tok8, r = r0 + (base + tile) * 16 + row16;
        if (tok < T && r < r1) {
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < kMainWarps; ++w) v += part[((w * C::CAP + tile) * NT + nt) * 128 + row16 * 8 + tok8];
          a.y[static_cast<int64_t>(tok) * a.H + r] = __float2bfloat16_rn(v + routed[tok * a.max_cols + (r - r0)]);
        }
      }
      bar_sync(1, kThr);
    }
    if (first) bar_sync(3, kDirThreads);
  }
}

// The router rows of a block, by the expert warps: K cut between the warps, sums through shared memory.
template <int NT>
__device__ __forceinline__ void router_rows(const DecodeArgs& a, float* part, const Share& b) {
  const int warp = (threadIdx.x >> 5) - kMainWarps, g = lane_id() >> 2, tid = threadIdx.x - 32 * kMainWarps;
  const int S = ceil_div(a.H, 32);
  const int s0 = S * warp / kExpWarps, s1 = S * (warp + 1) / kExpWarps;
  for (int base = b.n0; base < b.n1; base += 16) {
    const __nv_bfloat16* row[1][2];
    float acc[1][NT][4] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = base + 8 * h + g;
      row[0][h] = r >= b.n1 ? nullptr : (r < a.n ? a.kx + static_cast<int64_t>(r) * a.H : a.ky + static_cast<int64_t>(r - a.n) * a.H);
    }
    mma_rows<NT, 1, DirectCfg<NT>::D, false>(acc, row, a.x, a.T, a.H / 8, s0, s1);
    put_tile<NT>(part + warp * NT * 128, acc[0]);
    bar_sync(2, kExpThreads);
    for (int e = tid; e < NT * 128; e += kExpThreads) {
      const int row16 = e & 15, tok = e >> 4, r = base + row16;
      if (tok < a.T && r < b.n1) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kExpWarps; ++w) v += part[(w * NT + (tok >> 3)) * 128 + row16 * 8 + (tok & 7)];
        __stcg(a.logits + static_cast<int64_t>(tok) * (2 * a.n) + r, v);
      }
    }
    bar_sync(2, kExpThreads);
  }
  if (tid == 0) signal(a.counters + CNT_LOGITS);
}

template <int NT>
__global__ void __launch_bounds__(kDirThreads, 1) decode_direct_kernel(const DecodeArgs a) {
  extern __shared__ __align__(16) uint8_t smem_direct[];
  __shared__ ExpertShared s_exp;
  using C = DirectCfg<NT>;
  float* part = reinterpret_cast<float*>(smem_direct);
  uint8_t* scratch = smem_direct + C::kPartBytes;
  float* routed = reinterpret_cast<float*>(scratch + kScratchBytes);
  const Share b = share_of(a, blockIdx.x, gridDim.x);
  if (threadIdx.x < 32 * kMainWarps) {
    main_path<NT>(a, part, routed, b);
  } else {
    router_rows<NT>(a, reinterpret_cast<float*>(scratch), b);
    expert_path(a, s_exp, scratch, routed, b, kMainWarps);
    bar_arrive(3, kDirThreads);
  }
  __syncthreads();
  leave(a);
}

// ---- the ring form ----------------------------------------------------------------------------
// Warps by role: 0 producer (TMA boxes of weight rows and tokens into a ring of shared-memory slots), 1 tcgen05.mma with
// the weight rows as the M = 64 or 128 operand and the tokens as N = 16, 32 or 64, 2 - 5 epilogue, 6 - 13 experts.
// Weights do not depend on anything, so the producer runs ahead through router, gate / up and into the down projection
// until the ring is full, whatever the other roles wait for; only the token half of the first down slots is issued after
// the activation is complete.  A slot holds as many 64-wide K slices as fit, a slice the block's weight rows (128 bytes
// each, 128-byte swizzle) and the N token rows.  Rows of the tile beyond the block's own are whatever lies there; their
// accumulators are never read.
// A K slice costs the same four MMAs (23 to 48 cycles each) for 8 weight rows as for 128, and N token rows beside the
// weights.  Router and down projection have few rows a block, so there `rsplit` / `ksplit` blocks form a group that shares
// the group's rows and cuts K.  The partial logits are added by who selects; the partial sums of the down projection go
// through global memory to the block that owns the row, which adds them in block order.
template <int N>
__global__ void __launch_bounds__(kDecThreads, 1)
    decode_ring_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tkx, const __grid_constant__ CUtensorMap tky,
                  const __grid_constant__ CUtensorMap tg, const __grid_constant__ CUtensorMap tu, const __grid_constant__ CUtensorMap td,
                  const __grid_constant__ CUtensorMap ta, const DecodeArgs a) {
  using C = DecCfg<N>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ ExpertShared s_exp;
  __shared__ __align__(8) uint64_t s_bar[2 * kSlots + 6];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;  // swizzled tiles need 1024-byte alignment
  // ring | scratch of the expert warps | routed sums; the 128-row tile of the ring's last slice reads past its rows
  uint8_t* scratch = smem_raw + (base - raw) + a.slots * a.slot_bytes;
  float* routed = reinterpret_cast<float*>(scratch + kScratchBytes);
  Ring ring;
  ring.data = base, ring.full = smem_u32(s_bar), ring.empty = ring.full + 8 * kSlots;
  ring.abort_flag = &s_abort;
  const uint32_t acc_full = ring.full + 16 * kSlots, acc_free = acc_full + 32;
  const int warp = threadIdx.x >> 5;
  const int G = gridDim.x, c = blockIdx.x;
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < 2 * kSlots + 4; ++i) mbar_init(ring.full + 8 * i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(acc_free + 8 * i, kEpiWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tx), prefetch_tmap(&tkx), prefetch_tmap(&tky), prefetch_tmap(&tg), prefetch_tmap(&tu), prefetch_tmap(&td), prefetch_tmap(&ta);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&s_tmem), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const Share b = share_of(a, c, G);
  if (warp == 0) {
    if (elect_one()) producer<N>(a, ring, &tx, &tkx, &tky, &tg, &tu, &td, &ta, b);
  } else if (warp == 1) {
    if (elect_one()) mma_issuer<N>(a, ring, acc_full, acc_free, tmem, b);
  } else if (warp < kFirstExp) {
    epilogue<N>(a, ring, acc_full, acc_free, tmem, routed, b);
  } else {
    expert_path(a, s_exp, scratch, routed, b, kFirstExp);
    bar_sync(3, kFinalThreads);
    final_sums(a, routed, b, threadIdx.x - 64);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (s_abort) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies that are still on their way land before the block leaves
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
  leave(a);
}

int device_sms() {
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return v;
}

template <typename... KArgs, typename... Args>
int launch_cooperative(void (*kernel)(KArgs...), int blocks, int threads, size_t smem, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(-3, "few-token kernel: %s", cudaGetErrorString(e));
  }
  return 0;
}

template <int NT>
int launch_direct(DecodeArgs a, int sms, cudaStream_t st) {
  a.rsplit = a.ksplit = 1, a.rgroups = a.groups = sms;
  a.max_cols = 4 * ceil_div(a.H / 4, sms);
  const size_t smem = DirectCfg<NT>::kPartBytes + kScratchBytes + static_cast<size_t>(a.T) * a.max_cols * 4;
  static OncePerDevice once;
  if (once.first() && cudaFuncSetAttribute(decode_direct_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(-2, "cannot raise the shared-memory limit of decode_direct_kernel");
  }
  OMNI_REQUIRE(smem <= 160 * 1024, "hidden is too large for the few-token kernel on %d multiprocessors", sms);
  return launch_cooperative(decode_direct_kernel<NT>, sms, kDirThreads, smem, st, a);
}

template <int N>
int launch_ring(DecodeArgs a, int sms, cudaStream_t st) {
  a.rows_gu = ceil_div(a.I, sms) < 128 ? ceil_div(a.I, sms) : 128;
  // blocks of a group in the down projection: as many as its rows fit one tile, where K is long enough to cut (1 / 2 / 4
  // blocks: 24 tokens x 2048 x 5632 35.2 / 31.8 / 29.7 us, 64 x 2048 x 8192 50.8 / 42.6 / 40.3)
  a.ksplit = kMaxSplit;
  while (a.ksplit > 1 && (ceil_div(a.I, BK) < 8 * a.ksplit || 4 * ceil_div(a.H / 4, sms / a.ksplit) > BM || sms / a.ksplit > kMaxGroups)) a.ksplit /= 2;
  a.groups = sms / a.ksplit;
  a.rows_d = 4 * ceil_div(a.H / 4, a.groups);
  a.max_cols = 4 * ceil_div(ceil_div(a.H / 4, a.groups), a.ksplit);
  OMNI_REQUIRE(a.rows_d <= BM, "hidden is too large for the few-token kernel on %d multiprocessors", sms);
  // the same in the router, whose tile holds rows_r rows of each axis (a block at the border of the axes has both)
  a.rsplit = kMaxSplit;
  while (a.rsplit > 1 && (ceil_div(a.H, BK) < 2 * a.rsplit || 2 * round8(ceil_div(2 * a.n, sms / a.rsplit)) > BM)) a.rsplit /= 2;
  a.rgroups = sms / a.rsplit;
  a.rows_r = ceil_div(2 * a.n, a.rgroups);
  OMNI_REQUIRE(2 * round8(a.rows_r) <= BM, "sqrt_n is too large for the few-token kernel on %d multiprocessors", sms);
  a.m_r = 2 * round8(a.rows_r) <= 64 ? 64 : 128, a.m_gu = a.rows_gu <= 64 ? 64 : 128, a.m_d = a.rows_d <= 64 ? 64 : 128;
  const int slice_r = (2 * round8(a.rows_r) + N) * 128, slice_gu = (2 * round8(a.rows_gu) + N) * 128, slice_d = (round8(a.rows_d) + N) * 128;
  a.slot_bytes = kSlotBytes;
  for (int v : {slice_r, slice_gu, slice_d})
    if (a.slot_bytes < v) a.slot_bytes = v;
  a.slices_r = a.slot_bytes / slice_r, a.slices_gu = a.slot_bytes / slice_gu, a.slices_d = a.slot_bytes / slice_d;
  // behind the ring: at least the 16 KB that a 128-row tile at its end can reach over (the scratch alone is more)
  static_assert(kScratchBytes >= BM * 128, "slack behind the ring");
  const int tail = kScratchBytes + a.T * a.max_cols * 4;
  const int room = kSmemMost - 1024 - tail - static_cast<int>(sizeof(ExpertShared));
  a.slots = room / a.slot_bytes < kSlots ? room / a.slot_bytes : kSlots;
  OMNI_REQUIRE(a.slots >= 2, "hidden is too large for the few-token kernel");
  const size_t smem = 1024 + static_cast<size_t>(a.slots) * a.slot_bytes + tail;
  CUtensorMap tx, tkx, tky, tg, tu, td, ta;
  if (int e = tile_map(&tx, a.x, a.T, a.H, N)) return e;
  if (int e = tile_map(&tkx, a.kx, a.n, a.H, a.rows_r)) return e;
  if (int e = tile_map(&tky, a.ky, a.n, a.H, a.rows_r)) return e;
  if (int e = tile_map(&tg, a.wg, a.I, a.H, a.rows_gu)) return e;
  if (int e = tile_map(&tu, a.wu, a.I, a.H, a.rows_gu)) return e;
  if (int e = tile_map(&td, a.wd, a.H, a.I, a.rows_d)) return e;
  if (int e = tile_map(&ta, a.act, a.T, a.I, N)) return e;
  static OncePerDevice once;
  if (once.first() && cudaFuncSetAttribute(decode_ring_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           kSmemMost - static_cast<int>(sizeof(ExpertShared))) != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(-2, "cannot raise the shared-memory limit of decode_ring_kernel");
  }
  return launch_cooperative(decode_ring_kernel<N>, sms, kDecThreads, smem, st, tx, tkx, tky, tg, tu, td, ta, a);
}

// Blocks that work on one token's rows: as many as give each of a block's warps a row.
int share_of_token(int num_tokens, int k) {
  const int blocks = 148 / num_tokens, most = ceil_div(k, kExpWarps);
  return blocks < 1 ? 1 : (blocks < most ? blocks : most);
}
int64_t round16(int64_t v) { return (v + 15) & ~int64_t(15); }
bool is_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace omni

using namespace omni;

extern "C" int omni_decode_max_tokens(void) { return kDecMaxTokens; }

extern "C" size_t omni_decode_counter_bytes(void) { return CNT_WORDS * 4; }

extern "C" size_t omni_decode_workspace_bytes(int num_tokens, int hidden, int intermediate, int sqrt_n, int k) {
  if (num_tokens < 1 || num_tokens > kDecMaxTokens || hidden < 8 || intermediate < 8 || sqrt_n < 1 || k < 1) return 0;
  const int64_t T = num_tokens;
  return static_cast<size_t>(CNT_WORDS * 4 + round16(kMaxSplit * T * 2 * sqrt_n * 4) + share_of_token(num_tokens, k) * T * hidden * 4 +
                             round16(T * intermediate * 2) + kMaxSplit * T * hidden * 4);
}

extern "C" int omni_decode(const void* x, const void* gate_w, const void* up_w, const void* down_w, const void* router_x,
                           const void* router_y, const void* up_table, const void* down_table, const float* bn_scale,
                           const float* bn_shift, int num_tokens, int hidden, int intermediate, int sqrt_n, int k,
                           int64_t num_experts, void* y, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  OMNI_REQUIRE(num_tokens >= 0 && num_tokens <= kDecMaxTokens, "num_tokens must be in [0, %d], got %d", kDecMaxTokens, num_tokens);
  OMNI_REQUIRE(hidden >= 8 && hidden % 8 == 0, "hidden must be a positive multiple of 8, got %d", hidden);
  OMNI_REQUIRE(hidden <= 16384, "hidden must be at most 16384, got %d", hidden);
  OMNI_REQUIRE(intermediate >= 8 && intermediate % 8 == 0, "intermediate must be a positive multiple of 8, got %d", intermediate);
  OMNI_REQUIRE(sqrt_n >= 1 && sqrt_n <= 1024, "sqrt_n must be in [1, 1024], got %d", sqrt_n);
  OMNI_REQUIRE(k >= 1 && k <= kMaxK, "k must be in [1, %d], got %d", kMaxK, k);
  OMNI_REQUIRE(static_cast<int64_t>(k) <= static_cast<int64_t>(sqrt_n) * sqrt_n, "k = %d exceeds the %d experts", k, sqrt_n * sqrt_n);
  OMNI_REQUIRE(static_cast<int64_t>(sqrt_n) * sqrt_n <= num_experts, "the tables have %lld rows, the router selects among %d",
               static_cast<long long>(num_experts), sqrt_n * sqrt_n);
  OMNI_REQUIRE((bn_scale == nullptr) == (bn_shift == nullptr), "bn_scale and bn_shift must be given together");
  if (num_tokens == 0) return 0;
  OMNI_REQUIRE(x && gate_w && up_w && down_w && router_x && router_y && up_table && down_table && y && workspace && status, "NULL argument");
  OMNI_REQUIRE(is_aligned16(x) && is_aligned16(gate_w) && is_aligned16(up_w) && is_aligned16(down_w) && is_aligned16(router_x) &&
               is_aligned16(router_y) && is_aligned16(up_table) && is_aligned16(down_table) && is_aligned16(workspace),
               "pointers must be 16-byte aligned");
  const size_t need = omni_decode_workspace_bytes(num_tokens, hidden, intermediate, sqrt_n, k);
  OMNI_REQUIRE(workspace_bytes >= need, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const int sms = device_sms();
  OMNI_REQUIRE(sms > 0, "no CUDA device");
  DecodeArgs a{};
  const auto bf = [](const void* p) { return static_cast<const __nv_bfloat16*>(p); };
  a.x = bf(x), a.wg = bf(gate_w), a.wu = bf(up_w), a.wd = bf(down_w), a.kx = bf(router_x), a.ky = bf(router_y);
  a.up = bf(up_table), a.down = bf(down_table), a.bn_scale = bn_scale, a.bn_shift = bn_shift;
  a.T = num_tokens, a.H = hidden, a.I = intermediate, a.n = sqrt_n, a.k = k, a.kk = sqrt_n < k ? sqrt_n : k;
  a.cells = region_cells(a.kk, k);
  a.N = num_experts;
  a.share = share_of_token(num_tokens, k);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const int64_t T = num_tokens;
  a.counters = reinterpret_cast<int*>(w), w += CNT_WORDS * 4;
  a.logits = reinterpret_cast<float*>(w), w += round16(kMaxSplit * T * 2 * sqrt_n * 4);
  a.routed = reinterpret_cast<float*>(w), w += a.share * T * hidden * 4;
  a.act = reinterpret_cast<__nv_bfloat16*>(w), w += round16(T * intermediate * 2);
  a.partial = reinterpret_cast<float*>(w);
  a.y = static_cast<__nv_bfloat16*>(y), a.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // The form.  Up to 8 tokens the direct one is the faster at every size (8 tokens, hidden x intermediate, direct / ring in us:
  // 256 x 1024 13.6 / 17.6, 1024 x 4096 16.8 / 21.2, 2048 x 8192 30.3 / 32.3, 4096 x 11008 55.0 / 60.7).  From 9 to 16 it has
  // half the weights in flight and loses once a block has much to stream (16 tokens: 1024 x 4096, 0.17 MB a block, 18.7 / 21.2;
  // 2048 x 5632, 0.47 MB, 30.4 / 27.9; 4096 x 11008 72.1 / 62.5); beyond, its token operand no longer fits the registers.
  const int64_t bytes = 2 * (3 * static_cast<int64_t>(intermediate) + 2 * sqrt_n) * hidden;
  if (num_tokens <= 8) return launch_direct<1>(a, sms, st);
  if (num_tokens <= 16 && bytes <= sms * (int64_t(1) << 18)) return launch_direct<2>(a, sms, st);
  if (num_tokens <= 16) return launch_ring<16>(a, sms, st);
  if (num_tokens <= 32) return launch_ring<32>(a, sms, st);
  return launch_ring<64>(a, sms, st);
}
