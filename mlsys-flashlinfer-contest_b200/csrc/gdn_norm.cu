// Root-mean-square norm of rows with, optionally, the residual's addition in front, a
// SiLU gate before or after, and an e4m3 output with fp32 scales (sm_100a).
//
//   h = x (+ residual; h rounded once is residual_out) (* silu(gate) with gate_first)
//   y = h / sqrt(mean h^2 + eps) * weight (* silu(gate) without gate_first)
//   e4m3: scale = max |y| / 448 over the row or over each 128 columns (1 where that is
//   0), out = y / scale rounded to nearest (the quotient is fp32's: a value at a
//   rounding boundary goes where the formula puts it).
// h and y stay in fp32 from the loads to the one rounding of the output: the
// quantised values come from y itself, not from a 16-bit y, and the norm from the
// unrounded sum.
//
// Bound by HBM (one pass: every input is read once, kept in registers across the
// reduction).  A row belongs to kLanes threads, each holding kVecs 16-byte pieces.  16384 x 4096
// bf16 with residual to e4m3 by 128: 76 us, 0.95 of the copy peak; to bf16 81 us, 1.01; 245k heads of
// 128 with a gate 30 us, 0.94.
#include "gdn_internal.h"
#include "gdn_vec16.cuh"

namespace gdn {
namespace {

constexpr float kE4m3Max = 448.0f;
// Below this a scale's reciprocal, or the remainders of its quotients, would leave fp32's normal range:
// both sides of the quotient are lifted (exactly) first.
constexpr float kTinyScale = 0x1p-100f, kLift = 0x1p100f;

// The larger of the two, NaN if either is (a row that holds a NaN gets a NaN scale
// instead of hiding it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// Quotients by one divisor b, rounded to nearest, from r = 1 / b rounded to nearest: q = a r and one
// Newton step on it (Markstein, "Computation of elementary functions on the IBM RISC System/6000",
// IBM J. Res. Dev. 34, 1990), three operations.  For b and r in fp32's normal range; with b = +inf
// (r = 0) the step is made with 0, which leaves q as it is.  (Without the step a quotient is within 2 ulp,
// and a value near a rounding boundary lands a step of e4m3 away; 2.5 % of the time.  Two at a time in
// packed operations take 57 registers instead of 48, a block per SM less: +11 %.)
struct Divisor {
  float nb, r;
  __device__ __forceinline__ explicit Divisor(float b) {
    nb = b > 0x1.fffffep127f ? 0.f : -b;
    r = 1.0f / b;
  }
  __device__ __forceinline__ void divide(float& x, float& y) const {
    const float p = x * r, q = y * r;
    x = fmaf(fmaf(p, nb, x), r, p);
    y = fmaf(fmaf(q, nb, y), r, q);
  }
};

struct AddOp {
  static __device__ __forceinline__ float f(float a, float b) { return a + b; }
};
struct MaxOp {
  static __device__ __forceinline__ float f(float a, float b) { return max_nan(a, b); }
};

// Reduction over the kLanes threads of a row (every thread gets the result).  Rows of
// more than a warp go through shared memory; `slot` is a buffer no earlier reduction
// of this block used.
template <class Op, int kLanes>
__device__ __forceinline__ float row_reduce(float v, float* slot) {
#pragma unroll
  for (int d = 1; d < (kLanes < 32 ? kLanes : 32); d <<= 1)
    v = Op::f(v, __shfl_xor_sync(0xffffffffu, v, d));
  if constexpr (kLanes > 32) {
    constexpr int kWarps = kLanes / 32;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[warp] = v;
    __syncthreads();
    const float* mine = slot + warp / kWarps * kWarps;
    v = mine[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) v = Op::f(v, mine[i]);
  }
  return v;
}

enum GateMode { kNoGate = 0, kGateAfter = 1, kGateFirst = 2 };

template <class T, int kLanes, int kVecs, int kThreads, bool RESIDUAL, int GATE, bool FP8>
__global__ void __launch_bounds__(kThreads) gdn_rms_norm_kernel(NormArgs p) {
  constexpr int kRows = kThreads / kLanes;
  __shared__ float slots[2][kThreads / 32];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool live = row < p.rows;
  const int nvec = static_cast<int>(p.D >> 3);
  const uint16_t* x = static_cast<const uint16_t*>(p.x) + row * p.x_stride;
  const uint16_t* res = static_cast<const uint16_t*>(p.residual) + row * p.residual_stride;
  const uint16_t* gate = static_cast<const uint16_t*>(p.gate) + row * p.gate_stride;
  const uint16_t* weight = static_cast<const uint16_t*>(p.weight);

  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 xr[kVecs], rr[kVecs], gr[kVecs], wr[kVecs];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int i = lane + k * kLanes;
    const bool in = live && i < nvec;
    xr[k] = in ? ld_cs_u4(x + 8 * i) : zero;
    if (RESIDUAL) rr[k] = in ? ld_cs_u4(res + 8 * i) : zero;
    if (GATE != kNoGate) gr[k] = in ? ld_cs_u4(gate + 8 * i) : zero;
  }
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int i = lane + k * kLanes;
    wr[k] = i < nvec ? ldg_u4(weight + 8 * i) : zero;
  }

  float h[kVecs][8];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    unpack8<T>(xr[k], h[k]);
    if (RESIDUAL) {
      float r[8];
      unpack8<T>(rr[k], r);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[k][e] += r[e];
      const int i = lane + k * kLanes;
      if (live && i < nvec)
        st_u4(static_cast<uint16_t*>(p.residual_out) + row * p.D + 8 * i, pack8<T>(h[k]));
    }
    if (GATE == kGateFirst) {
      float g[8];
      unpack8<T>(gr[k], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[k][e] *= silu(g[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(h[k][e], h[k][e], ss);
  }
  ss = row_reduce<AddOp, kLanes>(ss, slots[0]);
  const float inv = 1.0f / sqrtf(ss / static_cast<float>(p.D) + p.eps);

  float amax = 0.f;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    float w[8];
    unpack8<T>(wr[k], w);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[k][e] *= inv * w[e];
    if (GATE == kGateAfter) {
      float g[8];
      unpack8<T>(gr[k], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[k][e] *= silu(g[e]);
    }
    if constexpr (!FP8) {
      const int i = lane + k * kLanes;
      if (live && i < nvec) st_u4(static_cast<uint16_t*>(p.out) + row * p.D + 8 * i, pack8<T>(h[k]));
    } else if (p.group == 0) {
      // (lanes past the row hold weight 0 and h 0, but 0 * inv is NaN where inv is not
      // finite; such a row is NaN anyway)
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = max_nan(amax, fabsf(h[k][e]));
    }
  }
  if constexpr (FP8) {
    if (p.group == 0) amax = row_reduce<MaxOp, kLanes>(amax, slots[1]);
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int i = lane + k * kLanes;
      if (p.group != 0) {  // 128 columns = 16 neighbouring lanes
        amax = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max_nan(amax, fabsf(h[k][e]));
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
      }
      // (a NaN maximum fails the comparison and stays)
      const float part = amax / kE4m3Max;
      const float scale = part == 0.f ? 1.f : part;
      if (live && i < nvec) {
        if (p.group != 0) {
          if ((i & 15) == 0) p.scale[row * (p.D >> 7) + (i >> 4)] = scale;
        } else if (i == 0) {
          p.scale[row] = scale;
        }
        float divisor = scale;
        if (scale < kTinyScale) {
          divisor *= kLift;
#pragma unroll
          for (int e = 0; e < 8; ++e) h[k][e] *= kLift;
        }
        const Divisor d(divisor);
#pragma unroll
        for (int e = 0; e < 8; e += 2) d.divide(h[k][e], h[k][e + 1]);
        uint2 q;
        q.x = e4m3x4(h[k][0], h[k][1], h[k][2], h[k][3]);
        q.y = e4m3x4(h[k][4], h[k][5], h[k][6], h[k][7]);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + row * p.D + 8 * i) = q;
      }
    }
  }
}

template <class T, int kLanes, int kVecs, int kThreads>
cudaError_t launch(const NormArgs& a, cudaStream_t s) {
  constexpr int kRows = kThreads / kLanes;
  const int64_t blocks = (a.rows + kRows - 1) / kRows;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned g = static_cast<unsigned>(blocks);
  const bool fp8 = a.scale != nullptr;
  const int gate = !a.gate ? kNoGate : a.gate_first ? kGateFirst : kGateAfter;
#define GDN_NORM(R, GATE, Q) gdn_rms_norm_kernel<T, kLanes, kVecs, kThreads, R, GATE, Q><<<g, kThreads, 0, s>>>(a)
  if (a.residual)
    fp8 ? GDN_NORM(true, kNoGate, true) : GDN_NORM(true, kNoGate, false);
  else if (gate == kGateFirst)
    fp8 ? GDN_NORM(false, kGateFirst, true) : GDN_NORM(false, kGateFirst, false);
  else if (gate == kGateAfter)
    fp8 ? GDN_NORM(false, kGateAfter, true) : GDN_NORM(false, kGateAfter, false);
  else
    fp8 ? GDN_NORM(false, kNoGate, true) : GDN_NORM(false, kNoGate, false);
#undef GDN_NORM
  return cudaGetLastError();
}

// Threads per row and their 16-byte pieces, as measured (us; more threads | these | fewer):
// 128 columns 30.4 with blocks of 128, 31.1 of 256, 32.4 of 512 (245k rows); 1024 columns 25.0 with
// 128 threads a row, 21.8 with a warp (no block-wide reduction; 32768 rows); 4096 columns, e4m3,
// 83.9 with 512, 74.2 with 256, 73.9 with 128; 8192: 96.7 with 1024, 87.2 with 512, 88.2 with 256;
// 16384: 96.6 with 1024, 80.8 with 512.  Eight rows of 4096 take 2.3-2.5 us with any of them.
template <class T>
cudaError_t by_size(const NormArgs& a, cudaStream_t s) {
  const int64_t v = a.D / 8;
  if (v <= 16) return launch<T, 16, 1, 128>(a, s);
  if (v <= 32) return launch<T, 32, 1, 256>(a, s);
  if (v <= 128) return launch<T, 32, 4, 128>(a, s);
  if (v <= 256) return launch<T, 256, 1, 256>(a, s);
  if (v <= 512) return launch<T, 256, 2, 256>(a, s);
  if (v <= 1024) return launch<T, 512, 2, 512>(a, s);
  return launch<T, 512, 4, 512>(a, s);
}

}  // namespace

cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t s) {
  return a.fp16 ? by_size<Fp16>(a, s) : by_size<Bf16>(a, s);
}

}  // namespace gdn
