// Short causal depthwise convolution: packed prompts, and tokens over a pool of
// convolution states (sm_100a).
//
// out[t, d] = act(bias[d] + sum_{j < W} w[d, j] x~[t - W + 1 + j, d]), where x~
// before a sequence's first token is the sequence's state (its last W - 1 inputs,
// oldest first) or zero.  The layer in front of a gated delta rule or a selective
// scan: its output columns go to up to four separate contiguous tensors (q | k | v
// or x | B | C), so that what follows needs no copy to make them contiguous.
//
// Bound by HBM: 2 W + ~6 operations per value against 4 bytes moved.  A thread owns
// eight neighbouring channels (one 16-byte access per row) and walks kTile tokens,
// keeping the window in registers, so each row is read once per tile plus W - 1 rows
// of the tile before; rows are loaded eight at a time before any is used.  Sums are in
// fp32, rounded once when stored; the states are copies of inputs (no arithmetic).
#include "gdn_internal.h"
#include "gdn_vec16.cuh"

namespace gdn {
namespace {

constexpr int kThreads = 128;  // 1024 channels per block

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

// Weights of eight channels ([D, W] row-major: 8 W contiguous values) and their bias.
template <class T, int W>
__device__ __forceinline__ void load_weights(const ConvParams& p, int64_t c0, float (&w)[W][8],
                                             float (&b)[8]) {
  float flat[8 * W];
#pragma unroll
  for (int i = 0; i < W; ++i) unpack8<T>(ldg_u4(p.weight + c0 * W + 8 * i), flat + 8 * i);
#pragma unroll
  for (int e = 0; e < 8; ++e)
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][e] = flat[e * W + j];
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = 0.f;
  if (p.bias) unpack8<T>(ldg_u4(p.bias + c0), b);
}

// One output row of eight channels from the window (W - 1 earlier rows, oldest
// first) and the current row.
template <class T, int W, bool SILU>
__device__ __forceinline__ uint4 conv_row(const float (&w)[W][8], const float (&b)[8],
                                          const float (&win)[W - 1][8], const float (&cur)[8]) {
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float acc = b[e];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) acc = fmaf(w[j][e], win[j][e], acc);
    acc = fmaf(w[W - 1][e], cur[e], acc);
    y[e] = SILU ? silu(acc) : acc;
  }
  return pack8<T>(y);
}

template <int W>
__device__ __forceinline__ void shift(float (&win)[W - 1][8], const float (&cur)[8]) {
#pragma unroll
  for (int j = 0; j < W - 2; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) win[j][e] = win[j + 1][e];
#pragma unroll
  for (int e = 0; e < 8; ++e) win[W - 2][e] = cur[e];
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

template <class T, int W, bool SILU, int kTile>
__global__ void __launch_bounds__(kThreads) gdn_conv_kernel(ConvParams p) {
  const int64_t c0 = (static_cast<int64_t>(blockIdx.x % p.col_blocks) * kThreads + threadIdx.x) * 8;
  const int64_t row = blockIdx.x / p.col_blocks;
  const bool mine = c0 < p.D;
  const int64_t tiles = (p.T + kTile - 1) / kTile;

  if (row >= tiles) {  // the new state of one sequence
    const int64_t n = row - tiles;
    const int64_t bos = min(max(p.cu[n], int64_t(0)), p.T);
    const int64_t eos = min(max(p.cu[n + 1], bos), p.T);
    if (!mine) return;
#pragma unroll
    for (int r = 0; r < W - 1; ++r) {
      const int64_t t = eos - (W - 1) + r;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (t >= bos)
        v = ldg_u4(p.x + t * p.x_row + c0);
      else if (p.state)
        v = ldg_u4(p.state + (n * (W - 1) + (t - bos) + W - 1) * p.D + c0);
      st_u4(p.new_state + (n * (W - 1) + r) * p.D + c0, v);
    }
    return;
  }

  const int64_t t0 = row * kTile;
  const int64_t t1 = min(t0 + kTile, p.T);
  // the sequence that holds t0 (or an earlier one that ends before it)
  const int64_t le = count_le(p.cu, p.N, t0);
  if (!mine) return;
  int64_t seq = min(le - 1, p.N - 1);  // -1: before the first sequence
  int64_t bos = seq >= 0 ? min(max(p.cu[seq], int64_t(0)), p.T) : 0;
  int64_t eos = seq >= 0 ? min(max(p.cu[seq + 1], bos), p.T) : min(max(p.cu[0], int64_t(0)), p.T);

  float w[W][8], b[8], win[W - 1][8];
  load_weights<T, W>(p, c0, w, b);
  const OutCol oc = out_col(p.out, c0);
  // the row before position t of sequence n (begin bos) as the window sees it
  auto before = [&](int64_t t, int64_t n, int64_t begin) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n >= 0) {
      if (t >= begin)
        v = ldg_u4(p.x + t * p.x_row + c0);
      else if (p.state && t >= begin - (W - 1))
        v = ldg_u4(p.state + (n * (W - 1) + (t - begin) + W - 1) * p.D + c0);
    }
    return v;
  };
#pragma unroll
  for (int j = 0; j < W - 1; ++j) unpack8<T>(before(t0 - (W - 1) + j, seq, bos), win[j]);

  for (int64_t tb = t0; tb < t1; tb += 8) {
    uint4 raw[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      raw[u] = tb + u < t1 ? ld_cs_u4(p.x + (tb + u) * p.x_row + c0) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t t = tb + u;
      if (t >= t1) break;
      while (t >= eos && seq + 1 < p.N) {  // the next sequence (empty ones are passed over)
        ++seq;
        bos = min(max(p.cu[seq], int64_t(0)), p.T);
        eos = min(max(p.cu[seq + 1], bos), p.T);
        if (t < eos) {
#pragma unroll
          for (int j = 0; j < W - 1; ++j) unpack8<T>(before(t - (W - 1) + j, seq, bos), win[j]);
        }
      }
      float cur[8];
      unpack8<T>(raw[u], cur);
      if (seq >= 0 && t >= bos && t < eos)
        st_u4(oc.base + t * oc.pitch, conv_row<T, W, SILU>(w, b, win, cur));
      shift<W>(win, cur);
    }
  }
}

// T tokens of one sequence per (block row, thread): the state rows and the first
// tokens are all loaded before any is used, and a thread writes only what it read.
template <class T, int W, bool SILU>
__global__ void __launch_bounds__(kThreads) gdn_conv_pool_kernel(ConvParams p) {
  const int64_t c0 = (static_cast<int64_t>(blockIdx.x % p.col_blocks) * kThreads + threadIdx.x) * 8;
  const int64_t n = blockIdx.x / p.col_blocks;
  if (c0 >= p.D) return;
  const int64_t in = p.in_slots[n];
  const int64_t outs = p.out_slots ? p.out_slots[n] : in;
  const uint16_t* xrow = p.x + n * p.x_batch + c0;
  float w[W][8], b[8], win[W - 1][8];
  uint4 st[W - 1];
  uint4 raw[4];
#pragma unroll
  for (int u = 0; u < 4; ++u)
    raw[u] = u < p.T ? ldg_u4(xrow + u * p.x_row) : make_uint4(0, 0, 0, 0);
  load_weights<T, W>(p, c0, w, b);
#pragma unroll
  for (int j = 0; j < W - 1; ++j)
    st[j] = in >= 0 && in < p.pool_size ? *reinterpret_cast<const uint4*>(p.pool + (in * (W - 1) + j) * p.D + c0)
                                        : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) unpack8<T>(st[j], win[j]);
  const OutCol oc = out_col(p.out, c0);
  for (int64_t tb = 0; tb < p.T; tb += 4) {
    if (tb > 0) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        raw[u] = tb + u < p.T ? ldg_u4(xrow + (tb + u) * p.x_row) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (tb + u >= p.T) break;
      float cur[8];
      unpack8<T>(raw[u], cur);
      st_u4(oc.base + (n * p.T + tb + u) * oc.pitch, conv_row<T, W, SILU>(w, b, win, cur));
      shift<W>(win, cur);
#pragma unroll
      for (int j = 0; j < W - 2; ++j) st[j] = st[j + 1];
      st[W - 2] = raw[u];
    }
  }
  if (outs >= 0 && outs < p.pool_size) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) st_u4(p.pool + (outs * (W - 1) + j) * p.D + c0, st[j]);
  }
}

constexpr int kTile = 32;

template <class T, int W, bool SILU>
cudaError_t launch(const ConvArgs& a, ConvParams p, cudaStream_t s) {
  p.col_blocks = static_cast<uint32_t>((a.D + kThreads * 8 - 1) / (kThreads * 8));
  const int64_t rows = a.in_slots ? a.N : (a.T + kTile - 1) / kTile + a.N;
  if (rows * p.col_blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(rows * p.col_blocks);
  if (a.in_slots)
    gdn_conv_pool_kernel<T, W, SILU><<<grid, kThreads, 0, s>>>(p);
  else
    gdn_conv_kernel<T, W, SILU, kTile><<<grid, kThreads, 0, s>>>(p);
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
                     0u, a.out};
  return a.fp16 ? by_width<Fp16>(a, p, s) : by_width<Bf16>(a, p, s);
}

}  // namespace gdn
