// Short causal depthwise convolution: packed prompts, and tokens over a pool of
// convolution states (sm_100a).
//
// out[t, d] = act(bias[d] + sum_{j < W} w[d, j] x~[t - W + 1 + j, d]), where x~
// before a sequence's first token is the sequence's state (its last W - 1 inputs,
// oldest first) or zero.  The layer in front of a gated delta rule or a selective
// scan: its output columns go to up to four separate contiguous tensors (q | k | v
// or x | B | C), so that what follows needs no copy to make them contiguous.
//
// Bound by HBM and, close behind, by the arithmetic units: 4 bytes moved a value against W
// products, 1.5 MUFU operations and ~6 others.  A thread owns eight neighbouring channels (one
// 16-byte access per row) and walks a run of tokens with the window in registers, so each row
// is read once per run plus W - 1 rows of the run before.  Rows ahead wait in shared memory
// (cp.async): held in registers, 8 at a time, they left room for 3 blocks per SM and 3.8 TB/s;
// like this 5.4-5.7 (bf16, W = 4: 7648 x 8192 in 47 us, 32768 x 6144 in 140 us; the copy peak
// gives 38 and 123).  Sums are in fp32, rounded once when stored; the states are copies of inputs.
#include <algorithm>

#include "gdn_internal.h"
#include "gdn_vec16.cuh"

namespace gdn {
namespace {

constexpr int kThreads = 128;   // 1024 channels per block
constexpr int kBlocksPerSm = 4;  // of the packed form: 128 registers a thread

struct ConvParams {
  const uint16_t* x;
  const uint16_t* weight;  // [D, W]
  const uint16_t* bias;    // [D] or nullptr
  const uint16_t* state;   // packed: [N, W-1, D] or nullptr
  uint16_t* new_state;     // packed: [N, W-1, D]
  uint16_t* pool;          // pool form: [pool_size, W-1, D]
  const int64_t* cu;
  const int32_t* in_slots;
  const int32_t* out_slots;
  int64_t x_batch, x_row;  // strides in elements
  int64_t T, N, D, pool_size;
  uint32_t col_blocks;  // blocks across the channels (fastest in the grid)
  int tile;             // packed: tokens of a block
  ConvOutputs out;
};

// The output tensor that holds channel c0 (a multiple of 8), and the row pitch and
// position in it.
struct OutCol {
  uint16_t* base;
  int64_t pitch;
};
__device__ __forceinline__ OutCol out_col(const ConvOutputs& o, int64_t c0) {
  OutCol r{static_cast<uint16_t*>(o.ptr[0]) + c0, o.width[0]};
  int64_t start = 0;
#pragma unroll
  for (int i = 1; i < kMaxConvOutputs; ++i) {
    if (i >= o.count) break;
    start += o.width[i - 1];
    if (c0 >= start) r = OutCol{static_cast<uint16_t*>(o.ptr[i]) + (c0 - start), o.width[i]};
  }
  return r;
}

// kCh neighbouring channels of a row (8 or 16 bytes).
template <int kCh>
struct Raw;
template <>
struct Raw<4> {
  uint2 v;
};
template <>
struct Raw<8> {
  uint4 v;
};
__device__ __forceinline__ void clear(Raw<4>& r) { r.v = make_uint2(0, 0); }
__device__ __forceinline__ void clear(Raw<8>& r) { r.v = make_uint4(0, 0, 0, 0); }
__device__ __forceinline__ void load(Raw<4>& r, const uint16_t* p) {
  asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(r.v.x), "=r"(r.v.y) : "l"(p));
}
__device__ __forceinline__ void load(Raw<8>& r, const uint16_t* p) {
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.v.x), "=r"(r.v.y), "=r"(r.v.z), "=r"(r.v.w)
               : "l"(p));
}
__device__ __forceinline__ void store(uint16_t* p, const Raw<4>& r) {
  asm volatile("st.global.v2.u32 [%0], {%1, %2};" ::"l"(p), "r"(r.v.x), "r"(r.v.y) : "memory");
}
__device__ __forceinline__ void store(uint16_t* p, const Raw<8>& r) { st_u4(p, r.v); }
template <class T>
__device__ __forceinline__ void unpack(const Raw<4>& r, float* f) {
  const float2 a = T::unpack(r.v.x), b = T::unpack(r.v.y);
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
}
template <class T>
__device__ __forceinline__ void unpack(const Raw<8>& r, float* f) {
  unpack8<T>(r.v, f);
}
template <class T>
__device__ __forceinline__ void pack(Raw<4>& r, const float* f) {
  r.v = make_uint2(T::pack(f[0], f[1]), T::pack(f[2], f[3]));
}
template <class T>
__device__ __forceinline__ void pack(Raw<8>& r, const float* f) {
  r.v = pack8<T>(f);
}

// Weights ([D, W] row-major: kCh W contiguous values) and bias of a thread's channels.
template <class T, int W, int kCh>
__device__ __forceinline__ void load_weights(const ConvParams& p, int64_t c0, float (&w)[W][kCh],
                                             float (&b)[kCh]) {
  float flat[kCh * W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    Raw<kCh> r;
    load(r, p.weight + c0 * W + kCh * i);
    unpack<T>(r, flat + kCh * i);
  }
#pragma unroll
  for (int e = 0; e < kCh; ++e)
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][e] = flat[e * W + j];
#pragma unroll
  for (int e = 0; e < kCh; ++e) b[e] = 0.f;
  if (p.bias) {
    Raw<kCh> r;
    load(r, p.bias + c0);
    unpack<T>(r, b);
  }
}

// silu x = x t^2 / (1 + t^2) with t = e^(x/2), for two values with one reciprocal: 1 / (a b) gives both,
// a = 1 + t^2.  MUFU operations bound the convolution next to HBM: three for two values instead of four.
// The exponents of t are held at 30, so that the product stays finite (the sigmoid is 1 there, to 2^-60);
// below, x t and t reach as far down as the type does, with neither clamp nor selection.  NaN and
// -inf give NaN, as in the formula, and fminf keeps a NaN to its own result.  (In scalar operations
// 3-5 % slower for prompts.)
__device__ __forceinline__ void silu2(float& x, float& y) {
  const float2 z = __fmul2_rn(make_float2(x, y), make_float2(0.5f * kLog2e, 0.5f * kLog2e));
  const float2 t = make_float2(ex2_ftz(fminf(z.x, 30.f)), ex2_ftz(fminf(z.y, 30.f)));
  const float2 a = __ffma2_rn(t, t, make_float2(1.f, 1.f));
  const float r = rcp_approx(a.x * a.y);
  const float2 v = __fmul2_rn(__fmul2_rn(make_float2(x, y), t), __fmul2_rn(t, __fmul2_rn(make_float2(r, r), make_float2(a.y, a.x))));
  x = v.x;
  y = v.y;
}

// One output row from the window (W - 1 earlier rows, oldest first) and the current row.
template <class T, int W, bool SILU, int kCh>
__device__ __forceinline__ Raw<kCh> conv_row(const float (&w)[W][kCh], const float (&b)[kCh],
                                             const float (&win)[W - 1][kCh], const float (&cur)[kCh]) {
  float y[kCh];
#pragma unroll
  for (int e = 0; e < kCh; e += 2) {
    float2 acc = make_float2(b[e], b[e + 1]);
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
      acc = __ffma2_rn(make_float2(w[j][e], w[j][e + 1]), make_float2(win[j][e], win[j][e + 1]), acc);
    acc = __ffma2_rn(make_float2(w[W - 1][e], w[W - 1][e + 1]), make_float2(cur[e], cur[e + 1]), acc);
    if (SILU) silu2(acc.x, acc.y);
    y[e] = acc.x;
    y[e + 1] = acc.y;
  }
  Raw<kCh> r;
  pack<T>(r, y);
  return r;
}

template <int W, int kCh>
__device__ __forceinline__ void shift(float (&win)[W - 1][kCh], const float (&cur)[kCh]) {
#pragma unroll
  for (int j = 0; j < W - 2; ++j)
#pragma unroll
    for (int e = 0; e < kCh; ++e) win[j][e] = win[j + 1][e];
#pragma unroll
  for (int e = 0; e < kCh; ++e) win[W - 2][e] = cur[e];
}

// 16 bytes global -> shared without registers; fewer `bytes` than 16 leave zeros.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// The number of entries of the non-decreasing cu[0..n] that are <= t, by a 32-way
// search: every warp lane tests one entry of each round (n + 1 <= 32: one load).
__device__ __forceinline__ int64_t count_le(const int64_t* cu, int64_t n, int64_t t) {
  int64_t lo = 0, len = n + 1;  // the answer lies in [lo, lo + len]
  const int lane = threadIdx.x & 31;
  while (len > 0) {
    const int64_t step = (len + 31) / 32;
    const int64_t i = lo + (lane + 1) * step - 1;  // last entry of this lane's part
    const bool le = i < lo + len && cu[i] <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    const int64_t end = lo + len;
    lo += c * step;
    len = min(step - 1, max(end - lo, int64_t(0)));
  }
  return lo;
}

// kBatch rows a step, kDepth steps of them in flight: each thread copies its own pieces of the
// rows ahead into its own places of shared memory (no barrier), where they cost no registers.
template <class T, int W, bool SILU, int kBatch, int kDepth>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) gdn_conv_kernel(ConvParams p) {
  constexpr int kCh = 8;
  using R = Raw<kCh>;
  __shared__ __align__(16) uint4 ring[kDepth][kBatch][kThreads];
  const int64_t c0 = (static_cast<int64_t>(blockIdx.x % p.col_blocks) * kThreads + threadIdx.x) * kCh;
  const int64_t row = blockIdx.x / p.col_blocks;
  const bool mine = c0 < p.D;
  const int64_t tiles = (p.T + p.tile - 1) / p.tile;

  if (row >= tiles) {  // the new state of one sequence
    const int64_t n = row - tiles;
    const int64_t bos = min(max(p.cu[n], int64_t(0)), p.T);
    const int64_t eos = min(max(p.cu[n + 1], bos), p.T);
    if (!mine) return;
#pragma unroll
    for (int r = 0; r < W - 1; ++r) {
      const int64_t t = eos - (W - 1) + r;
      R v;
      clear(v);
      if (t >= bos)
        load(v, p.x + t * p.x_row + c0);
      else if (p.state)
        load(v, p.state + (n * (W - 1) + (t - bos) + W - 1) * p.D + c0);
      store(p.new_state + (n * (W - 1) + r) * p.D + c0, v);
    }
    return;
  }

  const int64_t t0 = row * p.tile;
  const int rows = static_cast<int>(min(static_cast<int64_t>(p.tile), p.T - t0));
  const uint16_t* src = p.x + t0 * p.x_row + c0;
  auto fetch = [&](int r, int slot) {  // rows r.. (zeros past the tile)
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const bool in = mine && r + u < rows;
      cp_async16(&ring[slot][u][threadIdx.x], in ? src + (r + u) * p.x_row : p.x, in ? 16 : 0);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) fetch(d * kBatch, d);

  // the sequence that holds t0 (or an earlier one that ends before it; -1: before the first)
  const int64_t le = count_le(p.cu, p.N, t0);
  if (!mine) return;
  int64_t seq = min(le - 1, p.N - 1);
  int64_t bos = seq >= 0 ? min(max(p.cu[seq], int64_t(0)), p.T) : 0;
  int64_t eos = seq >= 0 ? min(max(p.cu[seq + 1], bos), p.T) : min(max(p.cu[0], int64_t(0)), p.T);
  // its rows of the tile, as [begin, end) from t0
  auto rel = [&](int64_t t) { return static_cast<int>(min(max(t - t0, int64_t(-W)), static_cast<int64_t>(p.tile))); };
  int begin = seq >= 0 ? rel(bos) : p.tile, end = rel(eos);

  float w[W][kCh], b[kCh], win[W - 1][kCh];
  load_weights<T, W, kCh>(p, c0, w, b);
  // the row at position t of sequence `seq` (begin `bos`) as the window sees it
  auto before = [&](int64_t t, float* f) {
    R v;
    clear(v);
    if (seq >= 0) {
      if (t >= bos)
        load(v, p.x + t * p.x_row + c0);
      else if (p.state && t >= bos - (W - 1))
        load(v, p.state + (seq * (W - 1) + (t - bos) + W - 1) * p.D + c0);
    }
    unpack<T>(v, f);
  };
#pragma unroll
  for (int j = 0; j < W - 1; ++j) before(t0 - (W - 1) + j, win[j]);
  const OutCol oc = out_col(p.out, c0);
  uint16_t* dst = oc.base + t0 * oc.pitch;

  int slot = 0;
  for (int r = 0; r < rows; r += kBatch) {
    cp_async_wait<kDepth - 2>();
    R raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) raw[u].v = ring[slot][u][threadIdx.x];
    fetch(r + (kDepth - 1) * kBatch, slot == 0 ? kDepth - 1 : slot - 1);  // (the slot used last)
    if (++slot == kDepth) slot = 0;
    if (r >= begin && r + kBatch <= end) {  // rows of one sequence
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        float cur[kCh];
        unpack<T>(raw[u], cur);
        store(dst, conv_row<T, W, SILU, kCh>(w, b, win, cur));
        dst += oc.pitch;
        shift<W, kCh>(win, cur);
      }
    } else {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (r + u >= rows) break;
        while (r + u >= end && seq + 1 < p.N) {  // the next sequence (empty ones are passed over)
          ++seq;
          bos = min(max(p.cu[seq], int64_t(0)), p.T);
          eos = min(max(p.cu[seq + 1], bos), p.T);
          begin = rel(bos);
          end = rel(eos);
          if (r + u < end) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) before(t0 + r + u - (W - 1) + j, win[j]);
          }
        }
        float cur[kCh];
        unpack<T>(raw[u], cur);
        if (r + u >= begin && r + u < end) store(dst, conv_row<T, W, SILU, kCh>(w, b, win, cur));
        dst += oc.pitch;
        shift<W, kCh>(win, cur);
      }
    }
  }
}

// T tokens of one sequence per (block row, thread): the state rows and the first
// tokens are all loaded before any is used, and a thread writes only what it read.
// Four channels a thread, kAhead tokens loaded at once: 256 x 4 tokens x 8192 channels in 15.0 us
// (eight channels: 15.9; kAhead 1: 19.0, 2: 18.4, 8: 17.8), 256 single tokens in 10.0 with kAhead 1
// (11.6 with 4; eight channels 10.6; two sequences a thread 9.8, but 2.1 for one sequence instead of
// 1.8), of which ~2 are the launch; the floors are 9 and 5.1.
template <class T, int W, bool SILU, int kCh, int kAhead>
__global__ void __launch_bounds__(kThreads) gdn_conv_pool_kernel(ConvParams p) {
  using R = Raw<kCh>;
  const int64_t c0 = (static_cast<int64_t>(blockIdx.x % p.col_blocks) * kThreads + threadIdx.x) * kCh;
  const int64_t n = blockIdx.x / p.col_blocks;
  if (c0 >= p.D) return;
  const int64_t in = p.in_slots[n];
  const int64_t outs = p.out_slots ? p.out_slots[n] : in;
  const uint16_t* xrow = p.x + n * p.x_batch + c0;
  float w[W][kCh], b[kCh], win[W - 1][kCh];
  R st[W - 1], raw[kAhead];
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      clear(raw[u]);
      if (t + u < p.T) load(raw[u], xrow + (t + u) * p.x_row);
    }
  };
  fetch(0);
  load_weights<T, W, kCh>(p, c0, w, b);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    clear(st[j]);
    if (in >= 0 && in < p.pool_size) load(st[j], p.pool + (in * (W - 1) + j) * p.D + c0);
  }
#pragma unroll
  for (int j = 0; j < W - 1; ++j) unpack<T>(st[j], win[j]);
  const OutCol oc = out_col(p.out, c0);
  for (int64_t tb = 0; tb < p.T; tb += kAhead) {
    if (tb > 0) fetch(tb);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (tb + u >= p.T) break;
      float cur[kCh];
      unpack<T>(raw[u], cur);
      store(oc.base + (n * p.T + tb + u) * oc.pitch, conv_row<T, W, SILU, kCh>(w, b, win, cur));
      shift<W, kCh>(win, cur);
#pragma unroll
      for (int j = 0; j < W - 2; ++j) st[j] = st[j + 1];
      st[W - 2] = raw[u];
    }
  }
  if (outs >= 0 && outs < p.pool_size) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store(p.pool + (outs * (W - 1) + j) * p.D + c0, st[j]);
  }
}

constexpr int kMinTile = 6, kBatch = 3, kDepth = 4, kCh = 8, kPoolCh = 4;

template <class T, int W, bool SILU>
cudaError_t launch(const ConvArgs& a, ConvParams p, cudaStream_t s) {
  const int ch = a.in_slots ? kPoolCh : kCh;
  p.col_blocks = static_cast<uint32_t>((a.D + kThreads * ch - 1) / (kThreads * ch));
  int64_t rows = a.N;
  if (!a.in_slots) {
    // One wave of blocks of equal length: a block's start (weights, its sequence, the rows before
    // it) costs as much as ~20 rows.
    const int64_t per_col = std::max<int64_t>(1, static_cast<int64_t>(device_sm_count()) * kBlocksPerSm / p.col_blocks);
    p.tile = static_cast<int>(std::min<int64_t>(std::max<int64_t>((a.T + per_col - 1) / per_col, kMinTile), 1 << 20));
    rows += (a.T + p.tile - 1) / p.tile;
  }
  if (rows * p.col_blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(rows * p.col_blocks);
  if (a.in_slots && a.T == 1)
    gdn_conv_pool_kernel<T, W, SILU, kPoolCh, 1><<<grid, kThreads, 0, s>>>(p);
  else if (a.in_slots)
    gdn_conv_pool_kernel<T, W, SILU, kPoolCh, 4><<<grid, kThreads, 0, s>>>(p);
  else
    gdn_conv_kernel<T, W, SILU, kBatch, kDepth><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

template <class T, int W>
cudaError_t by_act(const ConvArgs& a, const ConvParams& p, cudaStream_t s) {
  return a.silu ? launch<T, W, true>(a, p, s) : launch<T, W, false>(a, p, s);
}

template <class T>
cudaError_t by_width(const ConvArgs& a, const ConvParams& p, cudaStream_t s) {
  return a.W == 2 ? by_act<T, 2>(a, p, s) : a.W == 3 ? by_act<T, 3>(a, p, s) : by_act<T, 4>(a, p, s);
}

}  // namespace

cudaError_t launch_conv(const ConvArgs& a, cudaStream_t s) {
  const ConvParams p{static_cast<const uint16_t*>(a.x), static_cast<const uint16_t*>(a.weight),
                     static_cast<const uint16_t*>(a.bias), static_cast<const uint16_t*>(a.state),
                     static_cast<uint16_t*>(a.new_state), static_cast<uint16_t*>(a.pool), a.cu_seqlens,
                     a.in_slots, a.out_slots, a.x_batch_stride, a.x_row_stride, a.T, a.N, a.D, a.pool_size,
                     0u, 0, a.out};
  return a.fp16 ? by_width<Fp16>(a, p, s) : by_width<Bf16>(a, p, s);
}

}  // namespace gdn
