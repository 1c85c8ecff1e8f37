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
// operations).  A warp owns a batch of rows of one head; the lanes of a row hold 16 bytes of it
// each, so a warp's load covers whole 128-byte lines, and all of the batch's loads are in
// flight before the first is used.  The rows' dot products with C are reduced together: each
// exchange halves the values a lane still sums (9 shuffles for 8 rows instead of 40).  Gates
// are computed a token on a lane.  State and sums are fp32; a bf16 pool is rounded once per
// store.  Single tokens have their own instantiation, whose rows go from the raw load to the
// store one by one; with several, the rows stay in registers and two or four tokens' sums are reduced at
// once.  Measured with states larger than L2: single tokens, fp32, 256 x 64 heads of 64 x 128,
// 161 us (1.02 of the copy peak; 174 with two blocks per SM instead of three); bf16 84 us (0.99;
// 90 with three).  Four tokens, where the arithmetic counts: fp32 0.70, bf16 0.55.
#include "gdn_internal.h"
#include "gdn_vec16.cuh"

namespace gdn {
namespace {

constexpr int kWarps = 8;

// 16 bytes of state as loaded: four fp32 or eight bf16 elements
template <bool BF16>
__device__ __forceinline__ uint4 load_state(const void* base, int64_t elem) {
  return ld_cs_u4(static_cast<const uint8_t*>(base) + elem * (BF16 ? 2 : 4));
}
template <bool BF16>
__device__ __forceinline__ void widen(uint4 w, float2 (&s)[BF16 ? 4 : 2]) {
  if constexpr (BF16) {
    s[0] = Bf16::unpack(w.x);
    s[1] = Bf16::unpack(w.y);
    s[2] = Bf16::unpack(w.z);
    s[3] = Bf16::unpack(w.w);
  } else {
    s[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
    s[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
  }
}
template <bool BF16>
__device__ __forceinline__ void store_state(void* base, int64_t elem, const float2 (&s)[BF16 ? 4 : 2]) {
  uint4 v;
  if constexpr (BF16)
    v = make_uint4(pack_bf16x2(s[0].x, s[0].y), pack_bf16x2(s[1].x, s[1].y), pack_bf16x2(s[2].x, s[2].y),
                   pack_bf16x2(s[3].x, s[3].y));
  else
    v = make_uint4(__float_as_uint(s[0].x), __float_as_uint(s[0].y), __float_as_uint(s[1].x), __float_as_uint(s[1].y));
  asm volatile("st.global.cs.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(static_cast<uint8_t*>(base) + elem * (BF16 ? 2 : 4)),
               "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

// A lane's part of a B or C row (eight or four bf16), raw and widened
template <int kPairs>
struct Vec;
template <>
struct Vec<2> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  }
  __device__ __forceinline__ void widen(float2 (&f)[2]) const {
    f[0] = Bf16::unpack(v.x);
    f[1] = Bf16::unpack(v.y);
  }
};
template <>
struct Vec<4> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = ldg_u4(p); }
  __device__ __forceinline__ void widen(float2 (&f)[4]) const {
    f[0] = Bf16::unpack(v.x);
    f[1] = Bf16::unpack(v.y);
    f[2] = Bf16::unpack(v.z);
    f[3] = Bf16::unpack(v.w);
  }
};

// e^x, x <= 0, rounded to nearest where it is close to 1: a state that remembers thousands of tokens is
// multiplied by it as often, and what expf errs there, a quarter of a step to one side, adds up
// (4.6e-5 of the state after 3000 tokens of decay 1 - 3e-4, 1e-6 like this).
__device__ __forceinline__ float decay(float x) { return x > -0.5f ? 1.0f + expm1f(x) : expf(x); }

// kN bf16 values, kN = 4 or 8, widened
template <int kN>
__device__ __forceinline__ void widen_x(const Vec<kN / 2>& v, float (&x)[kN]) {
  float2 f[kN / 2];
  v.widen(f);
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    x[2 * i] = f[i].x;
    x[2 * i + 1] = f[i].y;
  }
}

// Ns = 64 or 128; BF16: storage of the state; PACKED: prompts by cu_seqlens (fp32 states
// in and out) instead of a pool; kTok: tokens whose inputs are loaded and whose sums are reduced
// together (1: each sequence has a single token); kU: rows a lane holds a part of.
template <int Ns, bool BF16, bool PACKED, int kTok, int kU, int kBlocks>
__global__ void __launch_bounds__(kWarps * 32, kBlocks) gdn_ssm_recurrent_kernel(SsmArgs p) {
  constexpr bool ONE = kTok == 1;
  constexpr int kVec = BF16 ? 8 : 4, kPairs = kVec / 2;
  constexpr int kLanes = Ns / kVec;        // lanes of a row: 8, 16 or 32
  constexpr int kRows = kU * 32 / kLanes;  // rows of a warp
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int per_head = static_cast<int>(p.P) / kRows;  // P is 64 or 128: a multiple of kRows
  const int64_t nh = unit / per_head;
  const int64_t n = nh / p.H;
  if (n >= p.N) return;
  const int h = static_cast<int>(nh - n * p.H);
  const int row0 = static_cast<int>(unit - nh * per_head) * kRows + lane / kLanes * kU;  // this lane's first row
  const int g = h / static_cast<int>(p.H / p.G);
  const int col = (lane % kLanes) * kVec;

  int64_t tok = 0;  // first token (a row of x, B, C, a, y) and their number
  int len = static_cast<int>(p.T);
  int64_t in = n, outs = n;
  if constexpr (PACKED) {
    tok = min(max(p.cu_seqlens[n], int64_t(0)), p.T);
    len = static_cast<int>(min(max(p.cu_seqlens[n + 1], tok), p.T) - tok);
  } else {
    tok = n * p.T;
    in = p.in_slots[n];
    outs = p.out_slots ? p.out_slots[n] : in;
  }
  const bool has_in = PACKED ? p.state != nullptr : in >= 0 && in < p.pool_size;
  const bool has_out = PACKED || (!p.no_state_update && outs >= 0 && outs < p.pool_size);
  const void* src = PACKED ? static_cast<const void*>(p.state) : p.pool;
  void* dst = PACKED ? static_cast<void*>(p.new_state) : p.pool;
  const int64_t src0 = ((in * p.H + h) * p.P + row0) * Ns + col;
  const int64_t dst0 = ((outs * p.H + h) * p.P + row0) * Ns + col;

  uint4 raw[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) raw[u] = has_in ? load_state<BF16>(src, src0 + u * Ns) : make_uint4(0, 0, 0, 0);

  const __nv_bfloat16* xs = static_cast<const __nv_bfloat16*>(p.x) + (tok * p.H + h) * p.P + row0;
  const __nv_bfloat16* bs = static_cast<const __nv_bfloat16*>(p.B) + (tok * p.G + g) * Ns + col;
  const __nv_bfloat16* cs = static_cast<const __nv_bfloat16*>(p.C) + (tok * p.G + g) * Ns + col;
  const __nv_bfloat16* as = static_cast<const __nv_bfloat16*>(p.a) + tok * p.H + h;
  __nv_bfloat16* ys = static_cast<__nv_bfloat16*>(p.out) + (tok * p.H + h) * p.P + row0;
  const int64_t xpitch = p.H * p.P, bpitch = p.G * Ns;

  // kTok tokens at a time: their inputs are loaded together, and their dot products reduced together
  Vec<kPairs> Bn[kTok], Cn[kTok];
  Vec<kU / 2> xn[kTok];
  auto inputs = [&](int t0) {
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const int64_t t = ONE ? 0 : min(t0 + i, len - 1);
      Bn[i].load(bs + t * bpitch);
      Cn[i].load(cs + t * bpitch);
      xn[i].load(xs + t * xpitch);
    }
  };
  if (ONE || len > 0) inputs(0);
  const float negA = -expf(p.A_log[h]);
  const float bias = p.dt_bias[h];
  const float skip = p.D ? p.D[h] : 0.f;
  float dts = 0.f, decs = 0.f;  // of token (t & ~31) + lane; with ONE of token 0
  auto gates = [&](int t) {
    dts = softplus_t20(__bfloat162float(as[t * p.H]) + bias);
    decs = decay(negA * dts);
  };
  if (ONE)
    gates(0);
  else if (lane < len)
    gates(lane);
  // Sums of kTok x kU values over the lanes of a row: every exchange halves the values that a
  // lane still sums; it ends with kLeft of them, the first of which is number `mine`.
  constexpr int kVals = kTok * kU, kLeft = kVals > kLanes ? kVals / kLanes : 1;
  int mine = 0;
#pragma unroll
  for (int half = kVals / 2, bit = kLanes / 2; half >= kLeft && bit >= 1; half >>= 1, bit >>= 1) mine |= lane & bit ? half : 0;
  const bool writer = kVals >= kLanes || (lane & (kLanes / kVals - 1)) == 0;
  auto reduce_and_write = [&](float (&acc)[kVals], int t0) {
#pragma unroll
    for (int half = kVals / 2, bit = kLanes / 2; half >= kLeft && bit >= 1; half >>= 1, bit >>= 1) {
      const bool up = lane & bit;
#pragma unroll
      for (int u = 0; u < half; ++u) {
        const float give = up ? acc[u] : acc[u + half];
        const float keep = up ? acc[u + half] : acc[u];
        acc[u] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
      }
    }
#pragma unroll
    for (int bit = kLanes / kVals / 2; bit >= 1; bit >>= 1) acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], bit);
#pragma unroll
    for (int i = 0; i < kLeft; ++i) {
      const int64_t at = (t0 + (mine + i) / kU) * xpitch + (mine + i) % kU;
      if (writer && (ONE || t0 + (mine + i) / kU < len))
        ys[at] = __float2bfloat16_rn(fmaf(skip, __bfloat162float(xs[at]), acc[i]));
    }
  };
  // one row's step: s <- dec s + w B; returns s . C over this lane's elements
  auto step = [&](float2 (&s)[kPairs], float w, float dec, const float2 (&B)[kPairs], const float2 (&C)[kPairs]) {
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      s[e] = __ffma2_rn(make_float2(dec, dec), s[e], __fmul2_rn(make_float2(w, w), B[e]));
      sum = __ffma2_rn(s[e], C[e], sum);
    }
    return sum.x + sum.y;
  };

  float acc[kVals];
  if constexpr (ONE) {
    float2 B[kPairs], C[kPairs];
    float xv[kU];
    Bn[0].widen(B);
    Cn[0].widen(C);
    widen_x<kU>(xn[0], xv);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float2 s[kPairs];
      widen<BF16>(raw[u], s);
      acc[u] = step(s, dts * xv[u], decs, B, C);
      if (has_out) store_state<BF16>(dst, dst0 + u * Ns, s);
    }
    reduce_and_write(acc, 0);
  } else {
    float2 s[kU][kPairs];
#pragma unroll
    for (int u = 0; u < kU; ++u) widen<BF16>(raw[u], s[u]);
#pragma unroll 1
    for (int t0 = 0; t0 < len; t0 += kTok) {
      if (t0 > 0) {
        if ((t0 & 31) == 0 && t0 + lane < len) gates(t0 + lane);
        inputs(t0);
      }
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        if (t0 + i < len) {
          const float dt = __shfl_sync(0xffffffffu, dts, (t0 + i) & 31), dec = __shfl_sync(0xffffffffu, decs, (t0 + i) & 31);
          float2 B[kPairs], C[kPairs];
          float xv[kU];
          Bn[i].widen(B);
          Cn[i].widen(C);
          widen_x<kU>(xn[i], xv);
#pragma unroll
          for (int u = 0; u < kU; ++u) acc[i * kU + u] = step(s[u], dt * xv[u], dec, B, C);
        } else {
#pragma unroll
          for (int u = 0; u < kU; ++u) acc[i * kU + u] = 0.f;
        }
      }
      reduce_and_write(acc, t0);
    }
    if (has_out) {
#pragma unroll
      for (int u = 0; u < kU; ++u) store_state<BF16>(dst, dst0 + u * Ns, s[u]);
    }
  }
}

template <int Ns, bool BF16, bool PACKED, int kTok, int kU, int kBlocks>
cudaError_t launch(const SsmArgs& a, cudaStream_t s) {
  constexpr int kRows = kU * 32 / (Ns / (BF16 ? 8 : 4));
  const int64_t units = a.N * a.H * (a.P / kRows);
  const int64_t blocks = (units + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  gdn_ssm_recurrent_kernel<Ns, BF16, PACKED, kTok, kU, kBlocks><<<static_cast<unsigned>(blocks), kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

// As measured (us; blocks per SM of single tokens: see above).  Two or four tokens at a time, bf16
// states, 128 x 32 heads of 128 x 128: 57 | 81 for two tokens, 71 | 86 for three, 78 | 92 for four,
// 132 | 150 for eight; fp32, 64 x 64 heads of 64 x 128: 48.5 | 53.5 for two, 58.2 | 55.9 for three,
// 62.0 | 59.1 for four, 95 | 86 for eight.  Four rows a lane instead of eight, with more blocks: up
// to 40 % slower.
template <int Ns>
cudaError_t by_form(const SsmArgs& a, cudaStream_t s) {
  if (!a.in_slots) return launch<Ns, false, true, 4, 8, 2>(a, s);
  if (a.state_bf16) return a.T == 1 ? launch<Ns, true, false, 1, 8, 2>(a, s) : launch<Ns, true, false, 2, 8, 2>(a, s);
  if (a.T <= 2) return a.T == 1 ? launch<Ns, false, false, 1, 8, 3>(a, s) : launch<Ns, false, false, 2, 8, 2>(a, s);
  return launch<Ns, false, false, 4, 8, 2>(a, s);
}

}  // namespace

cudaError_t launch_ssm_recurrent(const SsmArgs& a, cudaStream_t s) {
  return a.Ns == 64 ? by_form<64>(a, s) : by_form<128>(a, s);
}

}  // namespace gdn
