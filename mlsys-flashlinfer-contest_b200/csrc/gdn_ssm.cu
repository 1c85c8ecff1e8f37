// Selective state-space scan, token by token on CUDA cores (sm_100a): the pool form
// (T >= 1 tokens of each sequence of a decode batch) and short packed prompts.
//
// Per token and head, with dt = softplus(a + dt_bias) and one decay for the head:
//   S <- exp(-exp(A_log) dt) S + (dt x) B^T      [P, Ns]
//   y  = S C + D x
// S is the state after the token, in the k-last layout of the gated delta rule
// ([.., H, P, Ns]); head h reads B and C of group h / (H / G).
//
// Bound by the state's bytes (single tokens: 8 bytes an element in fp32 against ~4
// operations).  A warp owns kRows rows of one head; the lanes of a row hold 16 bytes of
// it each, so a warp's load covers whole 128-byte lines, and all of a warp's rows are in
// flight before the first is used.  The rows' dot products with C are reduced
// together: each exchange halves the values a lane still sums (9 shuffles for 8 rows
// instead of 40).  State and sums are fp32; a bf16 pool is rounded once per store.
#include "gdn_internal.h"
#include "gdn_vec16.cuh"

namespace gdn {
namespace {

constexpr int kWarps = 8;
constexpr int kU = 8;  // rows a lane holds a part of


template <bool BF16, int kVec>
__device__ __forceinline__ void load_state(const void* base, int64_t elem, float* s) {
  if constexpr (BF16) {
    unpack8<Bf16>(ld_cs_u4(static_cast<const uint16_t*>(base) + elem), s);
  } else {
    const float4 v = ld_stream_f4(static_cast<const float*>(base) + elem);
    s[0] = v.x;
    s[1] = v.y;
    s[2] = v.z;
    s[3] = v.w;
  }
}

template <bool BF16, int kVec>
__device__ __forceinline__ void store_state(void* base, int64_t elem, const float* s) {
  if constexpr (BF16) {
    const uint4 v = pack8<Bf16>(s);
    asm volatile("st.global.cs.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(static_cast<uint16_t*>(base) + elem),
                 "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
  } else {
    st_stream_f4(static_cast<float*>(base) + elem, make_float4(s[0], s[1], s[2], s[3]));
  }
}

// kVec consecutive bf16 values (8 or 16 bytes), widened
template <int kVec>
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float* v) {
  if constexpr (kVec == 8)
    unpack8<Bf16>(ldg_u4(p), v);
  else
    ld_bf16x4(p, v);
}

// Ns = 64 or 128; BF16: storage of the state; PACKED: prompts by cu_seqlens (fp32 states
// in and out) instead of a pool.
template <int Ns, bool BF16, bool PACKED>
__global__ void __launch_bounds__(kWarps * 32) gdn_ssm_recurrent_kernel(SsmArgs p) {
  constexpr int kVec = BF16 ? 8 : 4;
  constexpr int kLanes = Ns / kVec;        // lanes of a row: 8, 16 or 32
  constexpr int kPar = 32 / kLanes;        // rows of one warp access
  constexpr int kRows = kU * kPar;         // rows of a warp: 8, 16 or 32
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t per_head = p.P / kRows;    // P is 64 or 128: a multiple of kRows
  const int64_t n = unit / (p.H * per_head);
  if (n >= p.N) return;
  const int64_t hr = unit - n * p.H * per_head;
  const int64_t h = hr / per_head;
  const int64_t row0 = (hr - h * per_head) * kRows + lane / kLanes;  // + kPar u
  const int64_t g = h / (p.H / p.G);
  const int col = (lane % kLanes) * kVec;

  const __nv_bfloat16* xs = static_cast<const __nv_bfloat16*>(p.x);
  const __nv_bfloat16* bs = static_cast<const __nv_bfloat16*>(p.B);
  const __nv_bfloat16* cs = static_cast<const __nv_bfloat16*>(p.C);
  const __nv_bfloat16* as = static_cast<const __nv_bfloat16*>(p.a);
  __nv_bfloat16* ys = static_cast<__nv_bfloat16*>(p.out);

  int64_t tok = 0, len = p.T;  // first token (a row of x, B, C, a, y) and their number
  int64_t in = n, outs = n;
  if constexpr (PACKED) {
    tok = min(max(p.cu_seqlens[n], int64_t(0)), p.T);
    len = min(max(p.cu_seqlens[n + 1], tok), p.T) - tok;
  } else {
    tok = n * p.T;
    in = p.in_slots[n];
    outs = p.out_slots ? p.out_slots[n] : in;
  }
  const bool has_in = PACKED ? p.state != nullptr : in >= 0 && in < p.pool_size;
  const bool has_out = PACKED || (!p.no_state_update && outs >= 0 && outs < p.pool_size);
  const void* src = PACKED ? static_cast<const void*>(p.state) : p.pool;
  void* dst = PACKED ? static_cast<void*>(p.new_state) : p.pool;

  float s[kU][kVec];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    if (has_in)
      load_state<BF16, kVec>(src, ((in * p.H + h) * p.P + row0 + kPar * u) * Ns + col, s[u]);
    else
#pragma unroll
      for (int e = 0; e < kVec; ++e) s[u][e] = 0.f;
  }
  const float negA = -expf(p.A_log[h]);
  const float bias = p.dt_bias[h];
  const float skip = p.D ? p.D[h] : 0.f;
  // after the reduction lane l holds the sum of row kPar u + (its row group), u from
  // the lane bits that the exchanges below consumed
  const int ur = kLanes == 32 ? (lane >> 4 & 1) * 4 + (lane >> 3 & 1) * 2 + (lane >> 2 & 1)
                 : kLanes == 16 ? (lane >> 3 & 1) * 4 + (lane >> 2 & 1) * 2 + (lane >> 1 & 1)
                                : (lane >> 2 & 1) * 4 + (lane >> 1 & 1) * 2 + (lane & 1);
  constexpr int kSpare = kLanes / 8 - 1;  // lanes of the same row beyond the first
  const bool writer = (lane & kSpare) == 0;

  for (int64_t t = 0; t < len; ++t) {
    const int64_t r = tok + t;
    float B[kVec], C[kVec];
    load_vec<kVec>(bs + (r * p.G + g) * Ns + col, B);
    load_vec<kVec>(cs + (r * p.G + g) * Ns + col, C);
    const float dt = softplus_t20(__bfloat162float(as[r * p.H + h]) + bias);
    const float dec = expf(negA * dt);
    const __nv_bfloat16* xrow = xs + (r * p.H + h) * p.P + row0;
    float xv[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) xv[u] = __bfloat162float(xrow[kPar * u]);
    float acc[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const float w = dt * xv[u];
      acc[u] = 0.f;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        s[u][e] = fmaf(dec, s[u][e], w * B[e]);
        acc[u] = fmaf(s[u][e], C[e], acc[u]);
      }
    }
#pragma unroll
    for (int half = kU / 2, bit = kLanes / 2; half >= 1; half >>= 1, bit >>= 1) {
      const bool up = lane & bit;
#pragma unroll
      for (int u = 0; u < half; ++u) {
        const float give = up ? acc[u] : acc[u + half];
        const float keep = up ? acc[u + half] : acc[u];
        acc[u] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
      }
    }
#pragma unroll
    for (int bit = kLanes / 16; bit >= 1; bit >>= 1)
      acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], bit);
    float xo = xv[0];
#pragma unroll
    for (int u = 1; u < kU; ++u) xo = ur == u ? xv[u] : xo;
    if (writer)
      ys[(r * p.H + h) * p.P + row0 + kPar * ur] = __float2bfloat16_rn(fmaf(skip, xo, acc[0]));
  }
  if (has_out) {
#pragma unroll
    for (int u = 0; u < kU; ++u)
      store_state<BF16, kVec>(dst, ((outs * p.H + h) * p.P + row0 + kPar * u) * Ns + col, s[u]);
  }
}

template <int Ns, bool BF16, bool PACKED>
cudaError_t launch(const SsmArgs& a, cudaStream_t s) {
  constexpr int kRows = kU * 32 / (Ns / (BF16 ? 8 : 4));
  const int64_t units = a.N * a.H * (a.P / kRows);
  const int64_t blocks = (units + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  gdn_ssm_recurrent_kernel<Ns, BF16, PACKED><<<static_cast<unsigned>(blocks), kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_ssm_recurrent(const SsmArgs& a, cudaStream_t s) {
  if (!a.in_slots) return a.Ns == 64 ? launch<64, false, true>(a, s) : launch<128, false, true>(a, s);
  if (a.state_bf16) return a.Ns == 64 ? launch<64, true, false>(a, s) : launch<128, true, false>(a, s);
  return a.Ns == 64 ? launch<64, false, false>(a, s) : launch<128, false, false>(a, s);
}

}  // namespace gdn
