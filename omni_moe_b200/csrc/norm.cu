// Root-mean-square norm with the residual's addition, an optional 8-bit output with scales, and its gradient; and the
// conversion to and from MX blocks on its own.
//
//   h = x + r (rounded to the type)      rho = (mean_c h^2 + eps)^(-1/2)      y = h rho w      codes, scales = MX(y)
//   dz = dy w      dx = dr = rho (dz - h rho^2 mean_c(dz h)) + dh      dw_c = sum_t dy h rho
//
// Bound by bytes.  A row is read once: the threads of a row (one warp up to sixteen) hold it in registers, at most 32
// values each, add their partial sums by shuffles and, across warps, through shared memory.  All loads of a thread are
// issued before the first is used.  Sums are fp32.  The MX maximum of 32 neighbours is a shuffle among the lanes that
// hold them.  The codes are taken from the fp32 value of y, not from its rounded form.
//
// Gradient of the weight: a block walks over rows with a stride of the grid and keeps the sums of its columns in
// registers; one partial row per block goes to scratch and a second kernel adds the partial rows in block order (no
// atomics: run-to-run identical).
#include <type_traits>

#include "mx.cuh"
#include "tcgen05.cuh"

namespace omni {
namespace {

constexpr int kMaxHidden = 16384;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// VE neighbouring values moved by one instruction: 16 bytes, or a single value where a row's address or length does
// not allow more.
template <typename T, int VE>
struct __align__(sizeof(T) * VE < 16 ? sizeof(T) * VE : 16) Pack {
  T v[VE];
};
template <typename T, int VE>
__device__ __forceinline__ Pack<T, VE> load_pack(const T* p) {
  Pack<T, VE> r;
  if constexpr (VE * sizeof(T) == 16) *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  else if constexpr (VE * sizeof(T) == 32) {
    reinterpret_cast<uint4*>(&r)[0] = reinterpret_cast<const uint4*>(p)[0];
    reinterpret_cast<uint4*>(&r)[1] = reinterpret_cast<const uint4*>(p)[1];
  } else {
    static_assert(VE == 1, "one value or whole 16-byte pieces");
    r.v[0] = *p;
  }
  return r;
}
template <typename T, int VE>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VE>& r) {
  if constexpr (VE * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  else if constexpr (VE * sizeof(T) == 32) {
    reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<const uint4*>(&r)[0];
    reinterpret_cast<uint4*>(p)[1] = reinterpret_cast<const uint4*>(&r)[1];
  } else *p = r.v[0];
}

// Pieces to fp32 and back, two 16-bit values at a time: a bf16 is the upper half of an fp32, so unpacking is a shift and a
// mask, and one conversion packs two.  (Value by value the compiler spends a register and two instructions on each half.)
template <typename T, int VE>
__device__ __forceinline__ void unpack(const Pack<T, VE>& p, float (&f)[VE]) {
  if constexpr (sizeof(T) == 2 && VE % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&p);
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      float2 v;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) v = bf16x2_to_float2(w[i]);
      else v = __half22float2(*reinterpret_cast<const __half2*>(w + i));
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = to_f<T>(p.v[e]);
  }
}
template <typename T, int VE>
__device__ __forceinline__ Pack<T, VE> pack(const float (&f)[VE]) {
  Pack<T, VE> p;
  if constexpr (sizeof(T) == 2 && VE % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        w[i] = float2_to_bf16x2(f[2 * i], f[2 * i + 1]);
      } else {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) p.v[e] = from_f<T>(f[e]);
  }
  return p;
}

// w[c .. c + VE) as fp32, from a vector of the data's type or of fp32.
template <typename T, int VE>
__device__ __forceinline__ void load_weight(const void* w, bool w_f32, int c, float (&out)[VE]) {
  if (w_f32) {
    if constexpr (VE == 8) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(w) + c));
      const float4 b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(w) + c) + 1);
      out[0] = a.x, out[1] = a.y, out[2] = a.z, out[3] = a.w, out[4] = b.x, out[5] = b.y, out[6] = b.z, out[7] = b.w;
    } else if constexpr (VE == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(w) + c));
      out[0] = a.x, out[1] = a.y, out[2] = a.z, out[3] = a.w;
    } else {
      out[0] = __ldg(static_cast<const float*>(w) + c);
    }
  } else {
    unpack<T, VE>(load_pack<T, VE>(static_cast<const T*>(w) + c), out);
  }
}

// Sum over the threads of a row: `warps` warps, row group `grp` of the block.  Ends with all of them knowing it; the
// caller alternates `buf` between consecutive calls, so that no second barrier is needed.
__device__ __forceinline__ float row_sum(float v, int warps, int grp, int warp_in_row, float* buf) {
  v = warp_sum(v);
  if (warps == 1) return v;
  if (lane_id() == 0) buf[grp * 16 + warp_in_row] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < warps; ++i) s += buf[grp * 16 + i];
  return s;
}

// The scale's exponent of the MX block that this thread's VE values belong to.  All lanes of the warp call this; dead lanes
// pass zeros.  The maximum passes over NaN; an infinity in it sends the warp to the careful form.
template <int VE>
__device__ __forceinline__ int block_exponent(const float (&y)[VE]) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < VE; ++e) top = fmaxf(top, fabsf(y[e]));
#pragma unroll
  for (int o = 1; o < mx::kBlock / VE; o <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, o));
  if (__any_sync(FULL_MASK, top > 3.402823466e38f)) {
    top = 0.f;
#pragma unroll
    for (int e = 0; e < VE; ++e) top = fmaxf(top, mx::finite_abs(y[e]));
#pragma unroll
    for (int o = 1; o < mx::kBlock / VE; o <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, o));
  }
  return mx::exponent_of(top);
}
template <int VE>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&y)[VE], float inv) {
  if constexpr (VE == 8) *reinterpret_cast<uint2*>(p) = make_uint2(mx::encode4(y[0], y[1], y[2], y[3], inv), mx::encode4(y[4], y[5], y[6], y[7], inv));
  else if constexpr (VE == 4) *reinterpret_cast<uint32_t*>(p) = mx::encode4(y[0], y[1], y[2], y[3], inv);
  else *p = static_cast<uint8_t>(mx::encode2(y[0], 0.f, inv));
}

struct NormArgs {
  const void *x, *r, *w;
  int64_t ldx, ldr;
  int w_f32;
  int64_t T;
  int H;
  float eps;
  float shrink, grow;  // squares are added as f * (f * shrink), a power of two, so that a sum of squares that exceeds
                       // the range of fp32 has a mean that does not; mean = sum * grow
  int warps, rpc;  // warps of a row, rows of a block
  void *y, *h;     // h: null without a residual
  float* rstd;     // null unless kept for the gradient
  uint8_t *codes, *scales;  // null without the 8-bit output
};

template <typename T, int VE, int V>
__global__ void __launch_bounds__(512) rms_norm_kernel(const NormArgs a) {
  __shared__ float s_sum[8 * 16];
  const int tpr = a.warps * 32;
  const int grp = threadIdx.x / tpr, tid = threadIdx.x - grp * tpr;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * a.rpc + grp;
  const bool live = t < a.T;
  const T* x = static_cast<const T*>(a.x) + t * a.ldx;
  const T* r = static_cast<const T*>(a.r) + t * a.ldr;
  Pack<T, VE> px[V], pr[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * tpr + tid) * VE;
    if (live && c < a.H) px[i] = load_pack<T, VE>(x + c);
  }
  if (a.r) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * tpr + tid) * VE;
      if (live && c < a.H) pr[i] = load_pack<T, VE>(r + c);
    }
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * tpr + tid) * VE;
    if (live && c < a.H) {
      float f[VE];
      unpack<T, VE>(px[i], f);
      if (a.r) {
        float q[VE];
        unpack<T, VE>(pr[i], q);
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] += q[e];
        px[i] = pack<T, VE>(f);
        store_pack<T, VE>(static_cast<T*>(a.h) + t * a.H + c, px[i]);
        unpack<T, VE>(px[i], f);
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) sq = __fmaf_rn(f[e], f[e] * a.shrink, sq);
    }
  }
  sq = row_sum(sq, a.warps, grp, tid >> 5, s_sum);
  const float rho = rsqrtf(__fmaf_rn(sq, a.grow, a.eps));
  if (live && tid == 0 && a.rstd) a.rstd[t] = rho;
  const int scols = (a.H + mx::kBlock - 1) / mx::kBlock;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * tpr + tid) * VE;
    const bool in = live && c < a.H;
    float y[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) y[e] = 0.f;
    if (in) {
      float w[VE];
      load_weight<T, VE>(a.w, a.w_f32, c, w);
      unpack<T, VE>(px[i], y);
#pragma unroll
      for (int e = 0; e < VE; ++e) y[e] = y[e] * rho * w[e];
      store_pack<T, VE>(static_cast<T*>(a.y) + t * a.H + c, pack<T, VE>(y));
    }
    if (a.codes) {
      const int s = block_exponent<VE>(y);
      if (in) {
        store_codes<VE>(a.codes + t * a.H + c, y, mx::pow2(-s));
        if (c % mx::kBlock == 0) a.scales[t * scols + c / mx::kBlock] = static_cast<uint8_t>(s + 127);
      }
    }
  }
}

struct NormBwdArgs {
  const void *dy, *dh, *h, *w;
  int64_t lddy, lddh, ldh;
  const float* rstd;
  int w_f32;
  int64_t T;
  int H;
  float per_value;  // 1 / H
  int warps, rpc;
  void* dx;
  float* partial;  // [blocks, H] or null
  int32_t* status;
};

// The columns' sums of a block's row groups, added in group order.
template <int VE, int V>
__device__ __forceinline__ void put_partial(const NormBwdArgs& a, const float (&dw)[V][VE], float* s_dw, int tpr, int grp, int tid) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * tpr + tid) * VE;
    if (c < a.H) {
#pragma unroll
      for (int e = 0; e < VE; ++e) s_dw[grp * a.H + c + e] = dw[i][e];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
    float s = 0.f;
    for (int q = 0; q < a.rpc; ++q) s += s_dw[q * a.H + c];
    a.partial[static_cast<int64_t>(blockIdx.x) * a.H + c] = s;
  }
}

// One row, held by its threads: adds to their columns' sums and writes dx.
template <typename T, int VE, int V>
__device__ __forceinline__ void bwd_row(const NormBwdArgs& a, const Pack<T, VE> (&ph)[V], const Pack<T, VE> (&pg)[V], const Pack<T, VE> (&pd)[V],
                                        float rho, int64_t t, bool live, float (&dw)[V][VE], int tpr, int grp, int tid, float* s_sum) {
  float dot = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * tpr + tid) * VE;
    if (live && c < a.H) {
      float w[VE], h[VE], g[VE];
      load_weight<T, VE>(a.w, a.w_f32, c, w);
      unpack<T, VE>(ph[i], h), unpack<T, VE>(pg[i], g);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float n = h[e] * rho;
        dw[i][e] = __fmaf_rn(g[e], n, dw[i][e]);
        dot = __fmaf_rn(g[e] * w[e], n, dot);
      }
    }
  }
  dot = row_sum(dot, a.warps, grp, tid >> 5, s_sum) * a.per_value;
  const float back = -dot * rho * rho;  // rho (dz - h rho dot) = rho dz + h (-dot rho^2)
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * tpr + tid) * VE;
    if (live && c < a.H) {
      float w[VE], h[VE], g[VE];
      load_weight<T, VE>(a.w, a.w_f32, c, w);
      unpack<T, VE>(ph[i], h), unpack<T, VE>(pg[i], g);
#pragma unroll
      for (int e = 0; e < VE; ++e) g[e] = __fmaf_rn(h[e], back, rho * (g[e] * w[e]));
      if (a.dh) {
        unpack<T, VE>(pd[i], h);
#pragma unroll
        for (int e = 0; e < VE; ++e) g[e] += h[e];
      }
      store_pack<T, VE>(static_cast<T*>(a.dx) + t * a.H + c, pack<T, VE>(g));
    }
  }
}

// Rows straight into registers, one after the other: few rows, or rows that cannot be copied in 16-byte pieces.
template <typename T, int VE, int V>
__global__ void __launch_bounds__(512) rms_norm_bwd_kernel(const NormBwdArgs a) {
  __shared__ float s_sum[2 * 8 * 16];
  extern __shared__ __align__(16) uint8_t s_dyn[];
  const int tpr = a.warps * 32;
  const int grp = threadIdx.x / tpr, tid = threadIdx.x - grp * tpr;
  float dw[V][VE] = {};
  int turn = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.rpc;
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.rpc; t0 < a.T; t0 += step, turn ^= 1) {
    const int64_t t = t0 + grp;
    const bool live = t < a.T;
    Pack<T, VE> ph[V], pg[V], pd[V];
    const T* h = static_cast<const T*>(a.h) + t * a.ldh;
    const T* dy = static_cast<const T*>(a.dy) + t * a.lddy;
    const T* dh = static_cast<const T*>(a.dh) + t * a.lddh;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * tpr + tid) * VE;
      if (live && c < a.H) ph[i] = load_pack<T, VE>(h + c), pg[i] = load_pack<T, VE>(dy + c);
    }
    if (a.dh) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = (i * tpr + tid) * VE;
        if (live && c < a.H) pd[i] = load_pack<T, VE>(dh + c);
      }
    }
    bwd_row<T, VE, V>(a, ph, pg, pd, live ? a.rstd[t] : 0.f, t, live, dw, tpr, grp, tid, s_sum + turn * 128);
  }
  if (a.partial) put_partial<VE, V>(a, dw, reinterpret_cast<float*>(s_dyn), tpr, grp, tid);
}

// Many rows: the copy engine brings whole rows into a ring of shared-memory stages (rpc rows of h, dy and dh each), ahead
// of the threads, so that the barrier of a row's sum leaves no gap in the traffic.  (16384 x 4096 bf16 with dh: rows into
// registers 191 us, the next row's registers loaded ahead 140, ring 124, with two stages and a third block on the
// multiprocessor 97 = 5.5 TB/s; a producer warp of its own for the copies gains nothing.
// From kManyRows on: bf16, registers / ring, cold L2, in us: 1024 x 4096 22.9 / 21.5, 2048 x 4096 36 / 30, 4096 x 4096 54 / 40,
// at 256 and 1024 columns the same within 2; below, 512 x 256 11.3 / 13.3.  In fp32 the ring is the slower at 4096 columns, 66 / 79
// at 4096 rows, and the same within 2 at 256 and 1024.)
constexpr int kBwdStages = 2;
template <typename T, int VE, int V>
__global__ void __launch_bounds__(512) rms_norm_bwd_ring_kernel(const NormBwdArgs a) {
  __shared__ float s_sum[2 * 8 * 16];
  __shared__ __align__(8) uint64_t s_full[kBwdStages];
  __shared__ int s_abort;
  extern __shared__ __align__(16) uint8_t s_dyn[];  // stages of [3][rpc][H]; afterwards the row groups' column sums
  const int tpr = a.warps * 32;
  const int grp = threadIdx.x / tpr, tid = threadIdx.x - grp * tpr;
  const uint32_t full = tc::smem_u32(s_full);
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < kBwdStages; ++i) tc::mbar_init(full + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.rpc, first = static_cast<int64_t>(blockIdx.x) * a.rpc;
  const uint32_t row_bytes = a.H * sizeof(T);
  const int tensors = a.dh ? 3 : 2;
  const auto fetch = [&](int64_t t0, int stage) {  // one thread
    const int rows = static_cast<int>(a.T - t0 < a.rpc ? a.T - t0 : a.rpc);
    const uint32_t bar = full + 8 * stage;
    tc::mbar_arrive_expect_tx(bar, rows * tensors * row_bytes);
    for (int q = 0; q < tensors; ++q) {
      const T* src = static_cast<const T*>(q == 0 ? a.h : (q == 1 ? a.dy : a.dh));
      const int64_t ld = q == 0 ? a.ldh : (q == 1 ? a.lddy : a.lddh);
      for (int i = 0; i < rows; ++i)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                         tc::smem_u32(s_dyn) + ((stage * 3 + q) * a.rpc + i) * row_bytes),
                     "l"(src + (t0 + i) * ld), "r"(row_bytes), "r"(bar)
                     : "memory");
    }
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < kBwdStages; ++i)
      if (first + i * step < a.T) fetch(first + i * step, i);
  float dw[V][VE] = {};
  int turn = 0, stage = 0;
  uint32_t phase = 0;
  for (int64_t t0 = first; t0 < a.T; t0 += step, turn ^= 1) {
    const int64_t t = t0 + grp;
    const bool live = t < a.T;
    const float rho = live ? a.rstd[t] : 0.f;
    // a wait that runs out (a defect) flags it and leaves: every thread sees the flag after the barrier
    tc::mbar_wait(full + 8 * stage, phase, &s_abort, a.status);
    Pack<T, VE> ph[V], pg[V], pd[V];
    const T* base = reinterpret_cast<const T*>(s_dyn) + (static_cast<int64_t>(stage) * 3 * a.rpc + grp) * a.H;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * tpr + tid) * VE;
      if (live && c < a.H) {
        ph[i] = load_pack<T, VE>(base + c), pg[i] = load_pack<T, VE>(base + a.rpc * a.H + c);
        if (a.dh) pd[i] = load_pack<T, VE>(base + 2 * a.rpc * a.H + c);
      }
    }
    __syncthreads();  // the stage is read: it can be filled again
    if (s_abort) break;
    if (threadIdx.x == 0 && t0 + kBwdStages * step < a.T) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the reads above come before the copies' writes
      fetch(t0 + kBwdStages * step, stage);
    }
    if (++stage == kBwdStages) stage = 0, phase ^= 1;
    bwd_row<T, VE, V>(a, ph, pg, pd, rho, t, live, dw, tpr, grp, tid, s_sum + turn * 128);
  }
  if (s_abort) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies that are still on their way land before the block leaves
  }
  __syncthreads();
  if (a.partial) put_partial<VE, V>(a, dw, reinterpret_cast<float*>(s_dyn), tpr, grp, tid);
}

// dw[c] = the sum of the partial rows in block order: 32 columns x 32 slices of rows a block.
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* __restrict__ partial, int blocks, int H, void* dw, int dtype) {
  __shared__ float s_part[32][33];
  const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + col;
  float s = 0.f;
  if (c < H) {
#pragma unroll 4
    for (int b = slice; b < blocks; b += 32) s += partial[static_cast<int64_t>(b) * H + c];
  }
  s_part[slice][col] = s;
  __syncthreads();
  // warp w adds the 32 slices of column w, one in each lane
  const float v = warp_sum(s_part[col][slice]);
  const int wc = blockIdx.x * 32 + slice;
  if (col == 0 && wc < H) {
    const int c = wc;
    if (dtype == OMNI_F32) static_cast<float*>(dw)[c] = v;
    else if (dtype == OMNI_BF16) static_cast<__nv_bfloat16*>(dw)[c] = __float2bfloat16_rn(v);
    else static_cast<__half*>(dw)[c] = __float2half_rn(v);
  }
}

// MX blocks of a matrix: a thread has VE neighbours of one row, the lanes of a block of 32 share the maximum.  The
// columns of a row are padded to a whole number of warps' reach, so a block never crosses a warp or a row.
template <typename T, int VE>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int cols, uint8_t* codes,
                                                          uint8_t* scales) {
  const int scols = (cols + mx::kBlock - 1) / mx::kBlock;
  const int per_row = scols * (mx::kBlock / VE);  // threads of a row
  const int64_t total = rows * per_row;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  // whole warps stay in the loop together: the shuffles below need all lanes
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + (threadIdx.x & ~31); i0 < total; i0 += stride) {
    const int64_t i = i0 + lane_id();
    const int64_t t = i / per_row;
    const int c = static_cast<int>(i - t * per_row) * VE;
    const bool in = i < total && c < cols;
    float y[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) y[e] = 0.f;
    if (in) {
      const Pack<T, VE> p = load_pack<T, VE>(x + t * ldx + c);
#pragma unroll
      for (int e = 0; e < VE; ++e) y[e] = to_f<T>(p.v[e]);
    }
    const int s = block_exponent<VE>(y);
    if (in) {
      store_codes<VE>(codes + t * cols + c, y, mx::pow2(-s));
      if (c % mx::kBlock == 0) scales[t * scols + c / mx::kBlock] = static_cast<uint8_t>(s + 127);
    }
  }
}

// Decoded values: a thread has VE neighbours of a row (16: a 16-byte piece of codes), a block of threads walks along
// one row, the grid's second dimension over rows: no division.
template <typename T, int VE>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            int64_t rows, int cols, T* out) {
  const int scols = (cols + mx::kBlock - 1) / mx::kBlock;
  // (64 bits: the last threads of a row of almost 2^31 values lie behind it)
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * VE;
  if (c >= cols) return;
#pragma unroll 2
  for (int64_t t = static_cast<int64_t>(blockIdx.y) * blockDim.y + threadIdx.y; t < rows; t += static_cast<int64_t>(gridDim.y) * blockDim.y) {
    const uint8_t* p = codes + t * cols + c;
    const float sc = mx::scale_of(__ldg(scales + t * scols + c / mx::kBlock));
    if constexpr (VE == 16) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
      if constexpr (sizeof(T) == 2) {
        if ((reinterpret_cast<uintptr_t>(out) & 31) == 0) {  // 32 bytes in one store (two halves of a sector: 39 us instead)
          uint32_t o[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f0 = mx::decode2(w[e]), f1 = mx::decode2(w[e] >> 16);
            Pack<T, 4> v;
            v.v[0] = from_f<T>(f0.x * sc), v.v[1] = from_f<T>(f0.y * sc), v.v[2] = from_f<T>(f1.x * sc), v.v[3] = from_f<T>(f1.y * sc);
            o[2 * e] = reinterpret_cast<const uint32_t*>(&v)[0], o[2 * e + 1] = reinterpret_cast<const uint32_t*>(&v)[1];
          }
          asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + t * cols + c), "r"(o[0]), "r"(o[1]), "r"(o[2]),
                       "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                       : "memory");
          continue;
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        Pack<T, 8> o;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 f0 = mx::decode2(w[2 * half + e]), f1 = mx::decode2(w[2 * half + e] >> 16);
          o.v[4 * e] = from_f<T>(f0.x * sc), o.v[4 * e + 1] = from_f<T>(f0.y * sc);
          o.v[4 * e + 2] = from_f<T>(f1.x * sc), o.v[4 * e + 3] = from_f<T>(f1.y * sc);
        }
        store_pack<T, 8>(out + t * cols + c + 8 * half, o);
      }
    } else {
      out[t * cols + c] = from_f<T>(mx::decode2(*p).x * sc);
    }
  }
}

bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int multiprocessors() {
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1) return 148;
  return v;
}

// Threads of a row and rows of a block: `per_thread` values of a row in a thread (more only where sixteen warps would
// not reach the row's end), whole warps a row, about eight warps a block.
void row_shape(int64_t T, int H, int per_thread, int& per, int& warps, int& rpc) {
  per = per_thread;
  while (32 * 16 * per < H) per *= 2;  // 32 values reach kMaxHidden
  warps = ceil_div(H, 32 * per);
  rpc = warps >= 8 ? 1 : 8 / warps;
  if (T < rpc) rpc = static_cast<int>(T);
}
// Many rows: 16 values a thread; few rows: 8, so that a row's loads are spread over more warps.  (Forward with residual and
// codes, bf16, cold L2, 8 / 16 values in us: 16384 x 4096 117 / 97, 4096 x 4096 35.8 / 31.8, 2048 x 4096 22.4 / 19.4,
// 1024 x 4096 15.3 / 15.4, 512 x 1024 8.6 / 9.2, 256 x 1024 7.2 / 9.2.  At other widths, 256 to 8192, and in fp32 the two are
// within 2.5 us of one another, of 7 to 340, from 1024 rows on.)  Rows that move value by value need an address each: 8 as well.
constexpr int kManyRows = 1024;

template <typename T>
int launch_norm(const NormArgs& a0, cudaStream_t st) {
  NormArgs a = a0;
  constexpr int VE = 16 / sizeof(T);
  const bool vec = a.H % VE == 0 && at16(a.x) && at16(a.r) && at16(a.w) && at16(a.y) && at16(a.h) && at16(a.codes) &&
                   (a.ldx * sizeof(T)) % 16 == 0 && (a.ldr * sizeof(T)) % 16 == 0;
  int per;
  row_shape(a.T, a.H, vec && a.T >= kManyRows ? 16 : 8, per, a.warps, a.rpc);
  const int64_t blocks = ceil_div64(a.T, a.rpc);
  OMNI_REQUIRE(blocks < (int64_t(1) << 31), "too many rows");
  const dim3 grid(static_cast<unsigned>(blocks)), block(a.rpc * a.warps * 32);
  if (vec) {
    if (per == 8) rms_norm_kernel<T, VE, 8 / VE><<<grid, block, 0, st>>>(a);
    else if (per == 16) rms_norm_kernel<T, VE, 16 / VE><<<grid, block, 0, st>>>(a);
    else rms_norm_kernel<T, VE, 32 / VE><<<grid, block, 0, st>>>(a);
  } else {
    if (per == 8) rms_norm_kernel<T, 1, 8><<<grid, block, 0, st>>>(a);
    else if (per == 16) rms_norm_kernel<T, 1, 16><<<grid, block, 0, st>>>(a);
    else rms_norm_kernel<T, 1, 32><<<grid, block, 0, st>>>(a);
  }
  return check_launch("rms_norm_kernel");
}

// As many blocks as a multiprocessor holds at 80 registers a thread, which the ring's kernel has at 16 values of 16 bits
// (16384 x 4096 bf16, stages x blocks of 256 threads, before the packed conversions: 3 x 2 124 us, 2 x 2 113, 2 x 3 103),
// fewer where a block would have less than four turns (each costs a partial row).  Other instantiations are not as well
// served: at 16 values of 32 bits (112 registers) two of the three are resident, and from 6145 columns on a block has more
// than 384 threads, which leaves one.
constexpr int kBwdBlocks = 3;
int bwd_blocks(int64_t T, int rpc, int threads) {
  const int64_t turns = ceil_div64(T, rpc), sms = multiprocessors();
  const int per_sm = 256 * kBwdBlocks / threads < 1 ? 1 : (threads < 256 ? kBwdBlocks : 256 * kBwdBlocks / threads);
  int64_t blocks = turns / 4 < sms ? (turns < sms ? turns : sms) : turns / 4;
  if (blocks > per_sm * sms) blocks = per_sm * sms;
  return static_cast<int>(blocks);
}

template <typename T, int VE, int V>
int launch_bwd(const NormBwdArgs& a, int blocks, cudaStream_t st) {
  const size_t sums = a.partial ? sizeof(float) * a.rpc * a.H : 0;
  const dim3 block(a.rpc * a.warps * 32);
  if constexpr (VE > 1) {
    const size_t ring = static_cast<size_t>(kBwdStages) * 3 * a.rpc * a.H * sizeof(T);
    if (a.T >= kManyRows && ring <= 110 * 1024) {
      static OncePerDevice once;
      if (once.first() && cudaFuncSetAttribute(rms_norm_bwd_ring_kernel<T, VE, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, 110 * 1024) != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(-2, "cannot raise the shared-memory limit of rms_norm_bwd_ring_kernel");
      }
      rms_norm_bwd_ring_kernel<T, VE, V><<<blocks, block, ring > sums ? ring : sums, st>>>(a);
      return check_launch("rms_norm_bwd_ring_kernel");
    }
  }
  static OncePerDevice once;
  if (once.first() && cudaFuncSetAttribute(rms_norm_bwd_kernel<T, VE, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * kMaxHidden) != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(-2, "cannot raise the shared-memory limit of rms_norm_bwd_kernel");
  }
  rms_norm_bwd_kernel<T, VE, V><<<blocks, block, sums, st>>>(a);
  return check_launch("rms_norm_bwd_kernel");
}

template <typename T>
int bwd_for(NormBwdArgs a, void* dw, int dw_dtype, float* scratch, cudaStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  a.partial = dw ? scratch : nullptr;
  const bool vec = a.H % VE == 0 && at16(a.dy) && at16(a.dh) && at16(a.h) && at16(a.w) && at16(a.dx) && (a.lddy * sizeof(T)) % 16 == 0 &&
                   (a.lddh * sizeof(T)) % 16 == 0 && (a.ldh * sizeof(T)) % 16 == 0;
  int e, per;
  row_shape(a.T, a.H, vec && a.T >= kManyRows ? 16 : 8, per, a.warps, a.rpc);
  const int blocks = bwd_blocks(a.T, a.rpc, a.rpc * a.warps * 32);
  if (vec) e = per == 8 ? launch_bwd<T, VE, 8 / VE>(a, blocks, st) : per == 16 ? launch_bwd<T, VE, 16 / VE>(a, blocks, st) : launch_bwd<T, VE, 32 / VE>(a, blocks, st);
  else e = per == 8 ? launch_bwd<T, 1, 8>(a, blocks, st) : per == 16 ? launch_bwd<T, 1, 16>(a, blocks, st) : launch_bwd<T, 1, 32>(a, blocks, st);
  if (e) return e;
  if (dw) {
    norm_dw_kernel<<<ceil_div(a.H, 32), 1024, 0, st>>>(scratch, blocks, a.H, dw, dw_dtype);
    return check_launch("norm_dw_kernel");
  }
  return 0;
}

int check_norm(int dtype, int w_dtype, int64_t rows, int hidden) {
  OMNI_REQUIRE(dtype == OMNI_F32 || dtype == OMNI_BF16 || dtype == OMNI_F16, "unknown dtype %d", dtype);
  OMNI_REQUIRE(w_dtype == dtype || w_dtype == OMNI_F32, "the weight must have the data's type or float32");
  OMNI_REQUIRE(rows >= 0, "rows must be >= 0, got %lld", static_cast<long long>(rows));
  OMNI_REQUIRE(hidden >= 1 && hidden <= kMaxHidden, "hidden must be in [1, %d], got %d", kMaxHidden, hidden);
  return 0;
}

template <typename T>
int quantize_for(const void* x, int64_t ldx, int64_t rows, int cols, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  const int scols = ceil_div(cols, mx::kBlock);
  const bool vec = cols % VE == 0 && at16(x) && at16(codes) && (ldx * sizeof(T)) % 16 == 0;
  const int64_t threads = rows * scols * (mx::kBlock / (vec ? VE : 1));
  const int64_t want = ceil_div64(threads, 256), most = 16 * static_cast<int64_t>(multiprocessors());
  const unsigned grid = static_cast<unsigned>(want < most ? want : most);
  if (vec) mx_quantize_kernel<T, VE><<<grid, 256, 0, st>>>(static_cast<const T*>(x), ldx, rows, cols, codes, scales);
  else mx_quantize_kernel<T, 1><<<grid, 256, 0, st>>>(static_cast<const T*>(x), ldx, rows, cols, codes, scales);
  return check_launch("mx_quantize_kernel");
}

template <typename T>
int dequantize_for(const uint8_t* codes, const uint8_t* scales, int64_t rows, int cols, void* out, cudaStream_t st) {
  const bool vec = cols % 16 == 0 && at16(out) && at16(codes);
  const int pieces = ceil_div(cols, vec ? 16 : 1);
  int bx = 32;
  while (bx < pieces && bx < 256) bx *= 2;
  const dim3 block(bx, 256 / bx);
  const int64_t gx = ceil_div64(pieces, bx), want = ceil_div64(rows, 2 * block.y);
  OMNI_REQUIRE(gx < (int64_t(1) << 31), "too many columns");
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(want < 65535 ? want : 65535));
  if (vec) mx_dequantize_kernel<T, 16><<<grid, block, 0, st>>>(codes, scales, rows, cols, static_cast<T*>(out));
  else mx_dequantize_kernel<T, 1><<<grid, block, 0, st>>>(codes, scales, rows, cols, static_cast<T*>(out));
  return check_launch("mx_dequantize_kernel");
}

}  // namespace
}  // namespace omni

using namespace omni;

extern "C" int omni_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int w_dtype, int dtype,
                             int64_t rows, int hidden, float eps, void* y, void* h, float* rstd, void* codes, void* scales, void* stream) {
  if (int e = check_norm(dtype, w_dtype, rows, hidden)) return e;
  OMNI_REQUIRE(eps >= 0.f, "eps must be >= 0, got %g", static_cast<double>(eps));  // also refuses NaN
  OMNI_REQUIRE((residual == nullptr) == (h == nullptr), "residual and h must be given together");
  OMNI_REQUIRE((codes == nullptr) == (scales == nullptr), "codes and scales must be given together");
  if (rows == 0) return 0;
  OMNI_REQUIRE(x && weight && y, "NULL argument");
  OMNI_REQUIRE(rows == 1 || (ldx >= hidden && (!residual || ldr >= hidden)), "row strides must be at least hidden");
  NormArgs a{};
  a.x = x, a.r = residual, a.w = weight, a.ldx = ldx, a.ldr = residual ? ldr : 0, a.w_f32 = w_dtype == OMNI_F32;
  a.T = rows, a.H = hidden, a.eps = eps, a.y = y, a.h = h, a.rstd = rstd;
  int p = 1;
  while (p < hidden) p *= 2;
  a.shrink = 1.f / p, a.grow = static_cast<float>(p) / hidden;
  a.codes = static_cast<uint8_t*>(codes), a.scales = static_cast<uint8_t*>(scales);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == OMNI_F32) return launch_norm<float>(a, st);
  if (dtype == OMNI_BF16) return launch_norm<__nv_bfloat16>(a, st);
  return launch_norm<__half>(a, st);
}

extern "C" size_t omni_rms_norm_bwd_scratch_bytes(int64_t rows, int hidden) {
  if (rows < 1 || hidden < 1 || hidden > kMaxHidden) return 0;
  const int64_t most = kBwdBlocks * static_cast<int64_t>(multiprocessors());
  return sizeof(float) * static_cast<size_t>(rows < most ? rows : most) * hidden;
}

extern "C" int omni_rms_norm_bwd(const void* dy, int64_t lddy, const void* dh, int64_t lddh, const void* h, int64_t ldh, const void* weight,
                                 int w_dtype, int dtype, const float* rstd, int64_t rows, int hidden, void* dx, void* dweight,
                                 void* scratch, size_t scratch_bytes, int32_t* status, void* stream) {
  if (int e = check_norm(dtype, w_dtype, rows, hidden)) return e;
  if (rows == 0) return 0;
  OMNI_REQUIRE(dy && h && weight && rstd && dx && status, "NULL argument");
  OMNI_REQUIRE(rows == 1 || (lddy >= hidden && ldh >= hidden && (!dh || lddh >= hidden)), "row strides must be at least hidden");
  OMNI_REQUIRE(!dweight || (scratch && scratch_bytes >= omni_rms_norm_bwd_scratch_bytes(rows, hidden)), "the weight's gradient needs %zu bytes of scratch",
               omni_rms_norm_bwd_scratch_bytes(rows, hidden));
  NormBwdArgs a{};
  a.dy = dy, a.dh = dh, a.h = h, a.w = weight, a.lddy = lddy, a.lddh = dh ? lddh : 0, a.ldh = ldh, a.rstd = rstd;
  a.w_f32 = w_dtype == OMNI_F32, a.T = rows, a.H = hidden, a.per_value = 1.f / hidden, a.dx = dx, a.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* s = static_cast<float*>(scratch);
  if (dtype == OMNI_F32) return bwd_for<float>(a, dweight, w_dtype, s, st);
  if (dtype == OMNI_BF16) return bwd_for<__nv_bfloat16>(a, dweight, w_dtype, s, st);
  return bwd_for<__half>(a, dweight, w_dtype, s, st);
}

extern "C" int omni_mx_quantize(const void* x, int64_t ldx, int dtype, int64_t rows, int64_t cols, void* codes, void* scales, void* stream) {
  if (int e = check_norm(dtype, dtype, rows, 1)) return e;
  OMNI_REQUIRE(cols >= 1 && cols < (int64_t(1) << 31) - 64, "cols must be in [1, 2^31 - 64), got %lld", static_cast<long long>(cols));
  if (rows == 0) return 0;
  OMNI_REQUIRE(x && codes && scales, "NULL argument");
  OMNI_REQUIRE(rows == 1 || ldx >= cols, "the row stride must be at least cols");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t *q = static_cast<uint8_t*>(codes), *s = static_cast<uint8_t*>(scales);
  const int c = static_cast<int>(cols);
  if (dtype == OMNI_F32) return quantize_for<float>(x, ldx, rows, c, q, s, st);
  if (dtype == OMNI_BF16) return quantize_for<__nv_bfloat16>(x, ldx, rows, c, q, s, st);
  return quantize_for<__half>(x, ldx, rows, c, q, s, st);
}

extern "C" int omni_mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, int dtype, void* out, void* stream) {
  if (int e = check_norm(dtype, dtype, rows, 1)) return e;
  OMNI_REQUIRE(cols >= 1 && cols < (int64_t(1) << 31) - 64, "cols must be in [1, 2^31 - 64), got %lld", static_cast<long long>(cols));
  if (rows == 0) return 0;
  OMNI_REQUIRE(codes && scales && out, "NULL argument");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint8_t *q = static_cast<const uint8_t*>(codes), *s = static_cast<const uint8_t*>(scales);
  const int c = static_cast<int>(cols);
  if (dtype == OMNI_F32) return dequantize_for<float>(q, s, rows, c, out, st);
  if (dtype == OMNI_BF16) return dequantize_for<__nv_bfloat16>(q, s, rows, c, out, st);
  return dequantize_for<__half>(q, s, rows, c, out, st);
}
