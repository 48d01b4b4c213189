// The whole layer for a few tokens (1 <= T <= 64) in one kernel:
//   y[t] = (silu(x Wg^T) * (x Wu^T)) Wd^T + sum_{j<k} g_tj silu(x_t . Up[e_tj]) Down[e_tj]
// with (e, g) the router's product-key selection.  Every weight is used by T tokens only, so the kernel is bound by
// the bytes of Wg, Wu, Wd, the two sub-key matrices and the selected table rows, and by the latencies between its
// dependent parts.
//
// One persistent block per SM, launched cooperatively (its blocks wait on one another).  Every matrix is cut by rows:
// block c owns a contiguous range of gate / up columns, of router sub-keys and of output columns, so all blocks read
// the same number of bytes whatever the sizes, and no partial sum leaves a block.  Eight "main" warps stream the MLP,
// four "expert" warps do the router and the routed experts beside them:
//
//   main     gate | up rows -> act --[all act written]--> down rows -> + routed sum -> y
//   expert   router rows -> logits --[all logits written]--> selection, k dots (a few blocks per token)
//                                 --[all coefficients written]--> this block's columns of the k Down rows of every token
//
// The brackets are device-wide counters; a wait on one is bounded (status word).
//
// Dot products.  The weight rows are the A operand of mma.sync.m16n8k16 (16 rows), the tokens the B operand (8 tokens
// per n tile).  The contraction index may be permuted as long as both operands agree: lane (g, t) loads 16 contiguous
// bytes of row g (four lanes cover 64 bytes = two whole sectors) and uses its four words as fragments of two MMAs; the
// B words are the same 16 bytes of token g's row.  No staging, no shuffles; the warps of a block cut K between them and
// add their sums through shared memory in a fixed order.  Sums are fp32; act is rounded to bf16 (it is the B operand of
// the down projection), y once at the end.
#include <type_traits>

#include "router_select.cuh"

namespace omni {
namespace {

using namespace sel;

constexpr int kMainWarps = 8, kExpWarps = 4;
constexpr int kDecThreads = 32 * (kMainWarps + kExpWarps);
constexpr int kDecMaxTokens = 64;
// counters, one per 128-byte line
enum { CNT_LOGITS = 0, CNT_ACT = 32, CNT_COEF = 64, CNT_EXIT = 96, CNT_WORDS = 128 };

struct DecodeArgs {
  const __nv_bfloat16 *x, *wg, *wu, *wd, *kx, *ky, *up, *down;
  const float *bn_scale, *bn_shift;
  int T, H, I, n, k, kk, cells;
  int64_t N;
  int share;       // blocks that work on one token's dot products
  int max_cols;    // output columns of the widest block
  int* counters;
  float* logits;   // [T, 2n]
  float* coef;     // [T, k]
  int* index;      // [T, k]
  __nv_bfloat16* act;  // [T, I]
  __nv_bfloat16* y;
  int32_t* status;
};

template <int VPL, int CPL>
struct CoherentScratch : WarpScratch<VPL, CPL> {
  static constexpr bool kCoherent = true;  // the logits were written by other blocks of this launch
};

// Shapes of the main loops by token tiles (NT tiles of 8 tokens): TG weight tiles share the B fragments, D steps of 32
// along K are loaded before the first is used, CAP tiles are summed over the warps at a time.
template <int NT>
struct DecCfg {
  static constexpr int TG = NT >= 8 ? 1 : 2;
  static constexpr int D = NT <= 2 ? 4 : 2;
  static constexpr int CAP = NT == 1 ? 12 : (NT == 2 ? 8 : (NT == 4 ? 4 : 2));
  static constexpr int kPartBytes = kMainWarps * CAP * NT * 128 * 4;
  static constexpr int kRouterBytes = kExpWarps * NT * 128 * 4;
};

__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

__device__ __forceinline__ void signal(int* counter) {
  asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(counter) : "memory");
}
// Bounded: gives up after about two seconds, flags it, and lets the caller go on (its results are then invalid; every
// index that is read afterwards is checked before it is used as an address).
__device__ __forceinline__ void wait_for(const int* counter, int target, int32_t* status) {
  for (int i = 0; i < (1 << 22); ++i) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
    if (v >= target) return;
  }
  atomicOr(status, OMNI_ST_WAIT_TIMEOUT);
}

__device__ __forceinline__ uint4 ldg128_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 ldcg128(const void* p) { return __ldcg(reinterpret_cast<const uint4*>(p)); }

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
        b[d][nt] = in && tok < T ? (COHERENT ? ldcg128(p) : ldg128(p)) : zero;
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

// ---- main warps -------------------------------------------------------------------------------
template <int NT>
__device__ __forceinline__ void main_path(const DecodeArgs& a, float* part, const float* routed, int c0, int c1, int r0, int r1) {
  using C = DecCfg<NT>;
  const int warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2;
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
    __threadfence();
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
      if (first) bar_sync(3, kDecThreads);  // the expert warps have left the routed sums in shared memory
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
    if (first) bar_sync(3, kDecThreads);
  }
}

// ---- expert warps -----------------------------------------------------------------------------
template <int NT, int VPL, int CPL>
struct ExpertShared {
  CoherentScratch<VPL, CPL> sel;
  RegionTable region;
  float weight[kMaxK];
  int index[kMaxK];
};

template <int NT, int VPL, int CPL>
__device__ __forceinline__ void expert_path(const DecodeArgs& a, ExpertShared<NT, VPL, CPL>& sh, float* part, float* routed, int r0, int r1) {
  constexpr int kThr = 32 * kExpWarps;
  const int warp = (threadIdx.x >> 5) - kMainWarps, lane = lane_id(), g = lane >> 2;
  const int tid = threadIdx.x - 32 * kMainWarps;
  const int T = a.T, H8 = a.H / 8, k = a.k;
  const int G = gridDim.x, c = blockIdx.x;
  // router rows: sub-keys [q0, q1) of the 2n (x axis first)
  {
    const int S = ceil_div(a.H, 32);
    const int s0 = S * warp / kExpWarps, s1 = S * (warp + 1) / kExpWarps;
    const int q0 = static_cast<int>(static_cast<int64_t>(2 * a.n) * c / G), q1 = static_cast<int>(static_cast<int64_t>(2 * a.n) * (c + 1) / G);
    for (int base = q0; base < q1; base += 16) {
      const __nv_bfloat16* row[1][2];
      float acc[1][NT][4] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = base + 8 * h + g;
        row[0][h] = r >= q1 ? nullptr : (r < a.n ? a.kx + static_cast<int64_t>(r) * a.H : a.ky + static_cast<int64_t>(r - a.n) * a.H);
      }
      mma_rows<NT, 1, DecCfg<NT>::D, false>(acc, row, a.x, T, H8, s0, s1);
      put_tile<NT>(part + warp * NT * 128, acc[0]);
      bar_sync(2, kThr);
      for (int e = tid; e < NT * 128; e += kThr) {
        const int row16 = e & 15, tok = (e >> 4), r = base + row16;
        if (tok < T && r < q1) {
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < kExpWarps; ++w) v += part[(w * NT + (tok >> 3)) * 128 + row16 * 8 + (tok & 7)];
          a.logits[static_cast<int64_t>(tok) * (2 * a.n) + r] = v;
        }
      }
      bar_sync(2, kThr);
    }
    if (tid == 0) {
      __threadfence();
      signal(a.counters + CNT_LOGITS);
    }
  }
  // selection and dot products: `share` blocks per token, each selects (the same routing) and takes every share-th rank
  const int tasks = T * a.share;
  if (c < tasks) {
    if (tid == 0) wait_for(a.counters + CNT_LOGITS, G, a.status);
    bar_sync(2, kThr);
    TopkArgs s{};
    s.in_x = a.logits, s.ld_in = 2 * a.n, s.bn_scale = a.bn_scale, s.bn_shift = a.bn_shift;
    s.T = T, s.n = a.n, s.k = k, s.kk = a.kk, s.cells = a.cells;
    for (int task = c; task < tasks; task += G) {
      const int t = task / a.share, part_id = task - t * a.share;
      if (warp == 0) {
        uint32_t rkey[kMaxK / 32], rflat[kMaxK / 32];
        select_token<VPL, CPL, true>(s, t, sh.sel, sh.region.cell, rkey, rflat);
#pragma unroll
        for (int q = 0; q < kMaxK / 32; ++q) {
          const int r = q * 32 + lane;
          if (r < k) sh.weight[r] = expf(key_to_float(rkey[q])), sh.index[r] = static_cast<int>(rflat[q]);
        }
      }
      bar_sync(2, kThr);
      const uint4* xr = reinterpret_cast<const uint4*>(a.x + static_cast<int64_t>(t) * a.H);
      for (int j = part_id + a.share * warp; j < k; j += a.share * kExpWarps) {
        const int e = sh.index[j];
        float dot = 0.f;
        const bool ok = e >= 0 && e < a.N;
        if (ok) {
          const uint4* ur = reinterpret_cast<const uint4*>(a.up + static_cast<int64_t>(e) * a.H);
#pragma unroll 4
          for (int p = lane; p < H8; p += 32) {
            const uint4 u = ldg128_stream(ur + p), v = __ldg(xr + p);
            const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float2 uf = bf16x2_to_float2(uw[q]), vf = bf16x2_to_float2(vw[q]);
              dot = __fmaf_rn(uf.x, vf.x, dot), dot = __fmaf_rn(uf.y, vf.y, dot);
            }
          }
        }
        dot = warp_sum(dot);
        if (lane == 0) {
          if (!ok) atomicOr(a.status, OMNI_ST_BAD_EXPERT_INDEX);
          a.coef[static_cast<int64_t>(t) * k + j] = ok ? sh.weight[j] * silu(dot) : 0.f;
          a.index[static_cast<int64_t>(t) * k + j] = ok ? e : 0;
        }
      }
      bar_sync(2, kThr);
      if (tid == 0) {
        __threadfence();
        signal(a.counters + CNT_COEF);
      }
    }
  }
  // this block's output columns of the routed sum of every token: eight lanes share an item (token, 4 columns)
  if (tid == 0) wait_for(a.counters + CNT_COEF, tasks, a.status);
  bar_sync(2, kThr);
  const int quads = (r1 - r0) / 4;
  const int sub = lane & 7;
  for (int item0 = warp * 4; item0 < T * quads; item0 += kExpWarps * 4) {
    const int item = item0 + (lane >> 3);
    const bool live = item < T * quads;
    const int t = live ? item / quads : 0, col = r0 + (live ? item - t * quads : 0) * 4;
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
    if (live) {
#pragma unroll 4
      for (int j = sub; j < k; j += 8) {
        const float cf = __ldcg(a.coef + static_cast<int64_t>(t) * k + j);
        const int e = __ldcg(a.index + static_cast<int64_t>(t) * k + j);
        if (e >= 0 && e < a.N) {
          const uint2 d = __ldg(reinterpret_cast<const uint2*>(a.down + static_cast<int64_t>(e) * a.H + col));
          const float2 lo = bf16x2_to_float2(d.x), hi = bf16x2_to_float2(d.y);
          s0 = __fmaf_rn(cf, lo.x, s0), s1 = __fmaf_rn(cf, lo.y, s1), s2 = __fmaf_rn(cf, hi.x, s2), s3 = __fmaf_rn(cf, hi.y, s3);
        }
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      s0 += __shfl_xor_sync(FULL_MASK, s0, o), s1 += __shfl_xor_sync(FULL_MASK, s1, o);
      s2 += __shfl_xor_sync(FULL_MASK, s2, o), s3 += __shfl_xor_sync(FULL_MASK, s3, o);
    }
    if (live && sub == 0) {
      float* o = routed + t * a.max_cols + (col - r0);
      o[0] = s0, o[1] = s1, o[2] = s2, o[3] = s3;
    }
  }
}

template <int NT, int VPL, int CPL>
__global__ void __launch_bounds__(kDecThreads, 1) decode_kernel(const DecodeArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ ExpertShared<NT, VPL, CPL> s_exp;
  using C = DecCfg<NT>;
  float* part = reinterpret_cast<float*>(smem);
  float* rpart = reinterpret_cast<float*>(smem + C::kPartBytes);
  float* routed = reinterpret_cast<float*>(smem + C::kPartBytes + C::kRouterBytes);
  build_region_table(s_exp.region, a.kk, a.k, kMainWarps + kExpWarps);
  const int G = gridDim.x, c = blockIdx.x;
  const int c0 = static_cast<int>(static_cast<int64_t>(a.I) * c / G), c1 = static_cast<int>(static_cast<int64_t>(a.I) * (c + 1) / G);
  // output columns in groups of four: the Down rows are read in 8-byte pieces
  const int r0 = 4 * static_cast<int>(static_cast<int64_t>(a.H / 4) * c / G), r1 = 4 * static_cast<int>(static_cast<int64_t>(a.H / 4) * (c + 1) / G);
  if (threadIdx.x < 32 * kMainWarps) {
    main_path<NT>(a, part, routed, c0, c1, r0, r1);
  } else {
    expert_path<NT, VPL, CPL>(a, s_exp, rpart, routed, r0, r1);
    bar_arrive(3, kDecThreads);
  }
  __syncthreads();
  // the last block out leaves the counters as it found them: zero, for the next launch on this workspace
  if (threadIdx.x == 0) {
    __threadfence();
    if (atomicAdd(a.counters + CNT_EXIT, 1) == G - 1) {
      a.counters[CNT_LOGITS] = 0, a.counters[CNT_ACT] = 0, a.counters[CNT_COEF] = 0, a.counters[CNT_EXIT] = 0;
      __threadfence();
    }
  }
}

int device_sms() {
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return v;
}

template <int NT, int VPL, int CPL>
int launch_decode(DecodeArgs a, int sms, cudaStream_t st) {
  using C = DecCfg<NT>;
  const size_t smem = C::kPartBytes + C::kRouterBytes + static_cast<size_t>(a.T) * a.max_cols * 4;
  static OncePerDevice once;
  if (once.first() &&
      cudaFuncSetAttribute(decode_kernel<NT, VPL, CPL>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess)
    return fail(-2, "cannot raise the shared-memory limit of decode_kernel");
  OMNI_REQUIRE(smem <= 200 * 1024, "hidden is too large for the few-token kernel");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms), cfg.blockDim = dim3(kDecThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, decode_kernel<NT, VPL, CPL>, a);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(-3, "decode_kernel: %s", cudaGetErrorString(e));
  }
  return 0;
}

template <int NT>
int launch_nt(const DecodeArgs& a, int sms, cudaStream_t st) {
  if (a.n <= 64 && a.cells <= 64) return launch_decode<NT, 2, 2>(a, sms, st);
  if (a.n <= 256 && a.cells <= 320) return launch_decode<NT, 8, 10>(a, sms, st);
  return launch_decode<NT, 32, 22>(a, sms, st);
}

int64_t round16(int64_t v) { return (v + 15) & ~int64_t(15); }
bool is_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace omni

using namespace omni;

extern "C" int omni_decode_max_tokens(void) { return kDecMaxTokens; }

extern "C" size_t omni_decode_workspace_bytes(int num_tokens, int intermediate, int sqrt_n, int k) {
  if (num_tokens < 1 || num_tokens > kDecMaxTokens || intermediate < 8 || sqrt_n < 1 || k < 1) return 0;
  const int64_t T = num_tokens;
  return static_cast<size_t>(CNT_WORDS * 4 + round16(T * 2 * sqrt_n * 4) + 2 * round16(T * k * 4) + round16(T * intermediate * 2));
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
  const size_t need = omni_decode_workspace_bytes(num_tokens, intermediate, sqrt_n, k);
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
  // blocks per token for the dot products: enough that a block's four warps have one or two rows each
  a.share = sms / num_tokens;
  if (a.share > ceil_div(k, kExpWarps)) a.share = ceil_div(k, kExpWarps);
  if (a.share < 1) a.share = 1;
  a.max_cols = 4 * ceil_div(hidden / 4, sms);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const int64_t T = num_tokens;
  a.counters = reinterpret_cast<int*>(w), w += CNT_WORDS * 4;
  a.logits = reinterpret_cast<float*>(w), w += round16(T * 2 * sqrt_n * 4);
  a.coef = reinterpret_cast<float*>(w), w += round16(T * k * 4);
  a.index = reinterpret_cast<int*>(w), w += round16(T * k * 4);
  a.act = reinterpret_cast<__nv_bfloat16*>(w);
  a.y = static_cast<__nv_bfloat16*>(y), a.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (num_tokens <= 8) return launch_nt<1>(a, sms, st);
  if (num_tokens <= 16) return launch_nt<2>(a, sms, st);
  if (num_tokens <= 32) return launch_nt<4>(a, sms, st);
  return launch_nt<8>(a, sms, st);
}
