// Selective state-space scan of packed prompts in chunks of 64 tokens on tcgen05 tensor
// cores (sm_100a).
//
// A CTA owns 128 state rows of one sequence piece: two heads of 64 or one of 128, of one
// B/C group.  With gamma the inclusive cumulative log decay within the chunk and S [128, Ns]
// the state at its start, every accumulator is transposed (a TMEM lane is a state row
// (head, p)):
//   G      = C B^T                                  [i, j]    (one product for all heads)
//   M_h    = G e^{gamma_i - gamma_j} dt_j + D [i = j]  for j <= i      (bf16)
//   (M X)^T = X^T M^T,  (C S)^T = S C^T             [row, i]
//   y^T    = e^{gamma_i} (C S)^T + (M X)^T
//   S     <- e^{gamma_63} S + W^T B,   W = e^{gamma_63 - gamma_j} dt_j x_j
// Roundings: M and the S that C reads are bf16 operands (their errors, like the output's
// own rounding, are 2^-8 of a term).  The state itself stays fp32 in registers for the whole
// piece, and W enters its update as two bf16 terms (hi + lo, ~16 bits of mantissa; B is bf16
// already), so the fp32 final state keeps ~2^-17.
//
// The decays between a row and the columns of a 16-column block are r_i u_j with
// u_j = dt_j e^{gamma_top - gamma_j} (a table, top = the block's last column) and
// r_i = e^{gamma_i - gamma_top} below the diagonal; in blocks on the diagonal, where that
// could overflow, they are walked down each four columns from the highest j <= i.  No
// factor exceeds 1, whatever the decay.
//
// Values that are not finite stay where the recurrence puts them.  A masked factor 0 times
// an infinite x would leak into earlier tokens, and 0 times a NaN weight into the other
// head of a tile: x that is not finite is replaced by 0 as an operand and its row's outputs
// from that token on are set to NaN; gates that are not finite are 0 in the operands and NaN in
// the decays (e^gamma and the chunk's); tokens past the end are zeroed in x and B.
//
// Warp roles: warps 0-15 compute (four per TMEM lane quarter, each on a quarter of the
// columns), warp 16 issues the MMAs and the output's TMA stores, warp 17 the TMA loads.
// The compute warps run, for chunk c: the operands W (quarters 0-1) and M (quarters 2-3)
// of chunk c + 1, the outputs of chunk c, the state update of chunk c.  Each step's matrix
// products were issued a step earlier, so no step waits for one to run.
//
// Few (sequence, head tile) pairs: sequences are cut into pieces of `seg` tokens.  A first
// launch (STATE_ONLY) finds each piece's final state from zero and its decay; the second runs
// all pieces, each from S = decay S + F over the pieces before it.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <string.h>

#include "gdn_common.cuh"
#include "gdn_internal.h"
#include "gdn_sm100.cuh"

namespace gdn {

__device__ uint32_t g_ssm_status = 0;

namespace {
using namespace sm100;

constexpr int kComputeWarps = 16;
constexpr int kComputeThreads = 32 * kComputeWarps;
constexpr int kMmaWarp = 16;  // then the load warp
constexpr int kThreads = kComputeThreads + 64;
constexpr uint32_t kComputeBar = 1;
constexpr uint64_t kTimeoutNs = 2000000000ull;  // 2 s per wait, then give up
constexpr int kStages = 3;
constexpr int kRows = 128;  // state rows of a CTA

// ---- TMEM columns ----------------------------------------------------------
constexpr uint32_t TM_G = 0;     // lanes 64-127: G [i][j]
constexpr uint32_t TM_DS = 64;   // W^T B [row][n], two buffers of 128 columns
constexpr uint32_t TM_QS = 320;  // (C S)^T [row][i]
constexpr uint32_t TM_PV = 384;  // (M X)^T [row][i]
constexpr uint32_t TM_SB = 448;  // S as bf16 [row][n]: A operand
constexpr uint32_t kTmemCols = 512;

// ---- per-token tables (floats) of one head and chunk ------------------------
constexpr int G_GAM = 0;    // gamma, in log2 units
constexpr int G_D = 64;     // 2^(gamma_t - gamma_{t-1})
constexpr int G_DT = 128;   // dt (0 past the end)
constexpr int G_U = 192;    // dt 2^(gamma of the last token of t's 16 - gamma_t)
constexpr int G_W = 256;    // dt 2^(gamma_63 - gamma_t)
constexpr int G_EG = 320;   // 2^gamma_t
constexpr int kGateFloats = 384;
constexpr int kGateBufs = 3;

// ---- shared memory (offsets from a 1024-aligned base) ------------------------
template <int P, int NS>
struct Lay {
  static constexpr int kHeads = kRows / P;   // heads of a tile
  static constexpr int kKb = NS / 64;        // 64-column blocks of B and C
  static constexpr uint32_t kX = 16384;      // [block 2][t 64][128 B]
  static constexpr uint32_t kStage = kX + kKb * 16384;  // + [kb][B 64 rows | C 64 rows][128 B]
  static constexpr uint32_t OFF_Z0 = 0;      // 2 KiB of zeros below the stages ...
  static constexpr uint32_t OFF_ST = 2048;
  static constexpr uint32_t OFF_Z1 = OFF_ST + kStages * kStage;  // ... and above
  static constexpr uint32_t OFF_W = OFF_Z1 + 2048;    // W hi, then lo: [block 2][t 64][128 B]
  static constexpr uint32_t OFF_M = OFF_W + 32768;    // M of each head: [i 64][128 B]
  static constexpr uint32_t OFF_Y = OFF_M + 16384;    // outputs [block 2][t 64][128 B]
  static constexpr uint32_t OFF_G = OFF_Y + 16384;    // tables [buffer][head][kGateFloats]
  static constexpr uint32_t OFF_DEC = OFF_G + kGateBufs * 2 * kGateFloats * 4;  // [buffer][head]
  static constexpr uint32_t OFF_BAD = OFF_DEC + 32;   // first token whose x is not finite, by row
  static constexpr uint32_t OFF_BAR = OFF_BAD + kRows * 4;
  static constexpr uint32_t kBytes = OFF_BAR + 256 + 1024;
};
static_assert(Lay<64, 128>::kBytes <= 232448, "shared memory");

enum : int {
  B_FULL = 0,               // kStages: TMA loads landed
  B_EMPTY = B_FULL + kStages,  // kStages: every product that reads the stage is done
  B_RDY_W = B_EMPTY + kStages, B_RDY_M, B_RDY_D, B_RDY_S,  // compute warps -> issue warp
  B_G, B_DS, B_DS1, B_PV, B_QS, B_END, kNumBars            // products done
};

struct Params {
  const float* state;
  const float* A_log;
  const float* dt_bias;
  const float* D;
  const __nv_bfloat16* a;
  const int64_t* cu;
  __nv_bfloat16* out;
  float* new_state;
  float* ws;        // piece states in the compute threads' layout [slot][tile][128 NS]
  float* ws_dec;    // piece decays [slot][tile][2]
  int64_t T, N;
  int64_t seg;      // tokens of a piece (a multiple of 64); 0: sequences are whole
  int H, G, tiles;  // tiles: head tiles of all groups
};

__device__ __forceinline__ void load16(const float* src, float* v) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float4 x = reinterpret_cast<const float4*>(src)[q];
    v[4 * q] = x.x;
    v[4 * q + 1] = x.y;
    v[4 * q + 2] = x.z;
    v[4 * q + 3] = x.w;
  }
}

struct Piece {
  int64_t seq, bos, eos;  // sequence (-1: none) and the piece's tokens
  int index, count;       // of the sequence's pieces
};

// The piece of slot `slot`: sequences in order, each with max(1, ceil(length / seg)) pieces.
// Every warp finds it by itself, 32 sequences at a time.
__device__ __forceinline__ Piece find_piece(const Params& p, int64_t slot) {
  const int lane = threadIdx.x & 31;
  Piece r{-1, 0, 0, 0, 1};
  auto bounds = [&](int64_t n, int64_t* b, int64_t* e) {
    *b = min(max(p.cu[n], int64_t(0)), p.T);
    *e = min(max(p.cu[n + 1], *b), p.T);
  };
  if (p.seg == 0) {
    if (slot >= p.N) return r;
    r.seq = slot;
    bounds(slot, &r.bos, &r.eos);
    return r;
  }
  int64_t acc = 0;
  for (int64_t base = 0; base < p.N; base += 32) {
    const int64_t n = base + lane;
    int64_t b = 0, e = 0;
    int cnt = 0;
    if (n < p.N) {
      bounds(n, &b, &e);
      cnt = static_cast<int>(max(int64_t(1), (e - b + p.seg - 1) / p.seg));
    }
    int incl = cnt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, slot < acc + incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      r.seq = base + src;
      b = __shfl_sync(0xffffffffu, b, src);
      e = __shfl_sync(0xffffffffu, e, src);
      r.count = __shfl_sync(0xffffffffu, cnt, src);
      r.index = static_cast<int>(slot - acc) - (__shfl_sync(0xffffffffu, incl, src) - r.count);
      r.bos = b + r.index * p.seg;
      r.eos = min(r.bos + p.seg, e);
      return r;
    }
    acc += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}

template <int P, int NS, bool STATE_ONLY>
__global__ void __launch_bounds__(kThreads, 1)
    gdn_ssm_chunked_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_b,
                           const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ CUtensorMap tm_y,
                           const Params p) {
  using L = Lay<P, NS>;
  constexpr int kHeads = L::kHeads, kKb = L::kKb;
  constexpr int kCols = NS / 4;  // state columns of a compute thread
  constexpr int kWWarps = STATE_ONLY ? kComputeWarps : 8;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sb = smem_u32(smem);
  float* gates = reinterpret_cast<float*>(smem + L::OFF_G);
  float* decs = reinterpret_cast<float*>(smem + L::OFF_DEC);
  int* first_bad = reinterpret_cast<int*>(smem + L::OFF_BAD);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* any_bad = tmem_slot + 2;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = static_cast<int>(blockIdx.x % p.tiles);
  const int64_t slot = blockIdx.x / p.tiles;
  const int group_heads = p.H / p.G;
  const int group_tiles = p.tiles / p.G;
  const int g = tile / group_tiles;
  const int h0 = g * group_heads + (tile % group_tiles) * kHeads;  // first head of the tile
  const bool two = kHeads == 2 && h0 + 1 < (g + 1) * group_heads;  // its second head exists

  const Piece pc = find_piece(p, slot);
  if (pc.seq < 0 || (STATE_ONLY && pc.index == pc.count - 1)) return;
  const int64_t bos = pc.bos, Ltot = pc.eos - pc.bos;
  const bool last_piece = pc.index == pc.count - 1;
  const int n = static_cast<int>((Ltot + kChunk - 1) / kChunk);
  constexpr int64_t kHeadState = static_cast<int64_t>(P) * NS;

  // this thread's state rows and columns (compute warps)
  const int quarter = warp & 3, cq = (warp >> 2) & 3;
  const int row = 32 * quarter + lane;            // TMEM lane
  const int hh = kHeads == 2 ? row >> 6 : 0;      // head of the tile
  const bool row_live = hh == 0 || two;
  const int64_t row_off = (pc.seq * p.H + h0 + hh) * kHeadState + static_cast<int64_t>(row & (P - 1)) * NS + kCols * cq;

  if (Ltot <= 0) {  // an empty sequence keeps its state
    if (!STATE_ONLY && warp < kComputeWarps && row_live) {
#pragma unroll
      for (int i = 0; i < kCols / 4; ++i)
        st_stream_f4(p.new_state + row_off + 4 * i,
                     p.state ? ld_stream_f4(p.state + row_off + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f));
    }
    return;
  }

  if (tid == 0) {
    for (int i = 0; i < kNumBars; ++i)
      mbar_init(&bars[i], i == B_RDY_W ? kWWarps : i == B_RDY_M ? 8 : (i == B_RDY_D || i == B_RDY_S) ? kComputeWarps : 1);
    fence_mbar_init();
    *abort_flag = 0u;
    *any_bad = 0u;
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_b);
    if (!STATE_ONLY) {
      prefetch_tmap(&tm_c);
      prefetch_tmap(&tm_y);
    }
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  if (tid < kRows) first_bad[tid] = 0x7fffffff;
  if (!STATE_ONLY) {
    // zeros: the blocks beside the stages, M's columns above the diagonal
    for (int i = tid; i < 128; i += kThreads) {
      sts128(sb + L::OFF_Z0 + 16 * i, 0u, 0u, 0u, 0u);
      sts128(sb + L::OFF_Z1 + 16 * i, 0u, 0u, 0u, 0u);
    }
    for (int i = tid; i < 1024; i += kThreads) sts128(sb + L::OFF_M + 16 * i, 0u, 0u, 0u, 0u);
  }
  if (kHeads == 2 && !two)  // the absent head's x
    for (int i = tid; i < kStages * 512; i += kThreads)
      sts128(sb + L::OFF_ST + (i >> 9) * L::kStage + 8192 + 16 * (i & 511), 0u, 0u, 0u, 0u);
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool failed = false;

  if (warp < kComputeWarps) {
    // ======================= compute warps =================================
    const uint32_t tl = tmem + (static_cast<uint32_t>(quarter * 32) << 16);  // this warp's lanes
    auto signal = [&](int b, bool smem_written) {
      if (smem_written) fence_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[b]);
    };
    auto wait = [&](int b, uint32_t parity) {
      if (!failed) failed = !mbar_wait_nap(&bars[b], parity, kTimeoutNs);
      tc_fence_after();
    };
    auto table = [&](int c, int head) { return gates + ((c % kGateBufs) * 2 + head) * kGateFloats; };

    // ---- gates: warp 10 computes head 0's tables, warp 14 head 1's (quarter 2, the columns
    //      of M above the diagonal, where there is nothing else to do) ---------------
    const bool gate_warp = quarter == 2 && (cq == 2 || (cq == 3 && kHeads == 2));
    const int gh = cq - 2;
    const bool gate_live = gate_warp && (gh == 0 || two);
    float negA = 0.f, bias = 0.f;
    unsigned short raw[2] = {0, 0};
    if (gate_live) {
      negA = -expf(p.A_log[h0 + gh]) * kLog2e;
      bias = p.dt_bias[h0 + gh];
    }
    auto prefetch_gates = [&](int c) {
      if (!gate_live) return;
      const unsigned short* pa = reinterpret_cast<const unsigned short*>(p.a);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t t = bos + static_cast<int64_t>(c) * kChunk + 2 * lane + e;
        if (t < pc.eos) raw[e] = pa[t * p.H + h0 + gh];
      }
    };
    auto compute_gates = [&](int c) {
      const int Lc = gate_live ? static_cast<int>(min(static_cast<int64_t>(kChunk), Ltot - static_cast<int64_t>(c) * kChunk)) : 0;
      float dt[2], lg[2];
      bool ok[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool valid = 2 * lane + e < Lc;
        dt[e] = valid ? softplus_t20(bf16_bits_to_f32(raw[e]) + bias) : 0.f;
        lg[e] = valid ? negA * dt[e] : 0.f;
        ok[e] = dt[e] < __int_as_float(0x7f800000) && lg[e] == lg[e];
        // 2^-256 is 0 in fp32: a stronger decay is the same, and sums stay finite
        lg[e] = ok[e] ? fmaxf(lg[e], -256.f) : 0.f;
        dt[e] = ok[e] ? dt[e] : 0.f;
      }
      const unsigned bad0 = __ballot_sync(0xffffffffu, !ok[0]), bad1 = __ballot_sync(0xffffffffu, !ok[1]);
      const int fb = min(bad0 ? 2 * (__ffs(bad0) - 1) : 64, bad1 ? 2 * (__ffs(bad1) - 1) + 1 : 64);
      const float pair = lg[0] + lg[1];
      float incl = pair, suf = pair;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const float y = __shfl_up_sync(0xffffffffu, incl, d);
        const float z = __shfl_down_sync(0xffffffffu, suf, d);
        if (lane >= d) incl += y;
        if (lane + d < 32) suf += z;
      }
      const float gt[2] = {incl - lg[1], incl};
      // gamma_63 - gamma_t as a sum of its own terms (a difference of two long sums would lose
      // the weights' precision where the decay is strong)
      const float after = __shfl_down_sync(0xffffffffu, suf, 1);
      const float tail1 = lane == 31 ? 0.f : after;
      const float rest[2] = {tail1 + lg[1], tail1};
      const float top = __shfl_sync(0xffffffffu, gt[1], lane | 7);
      const float g63 = __shfl_sync(0xffffffffu, gt[1], 31);
      float* tb = table(c, gh);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 2 * lane + e;
        tb[G_GAM + t] = gt[e];
        tb[G_D + t] = ex2_ftz(lg[e]);
        tb[G_DT + t] = dt[e];
        tb[G_U + t] = dt[e] * ex2_ftz(top - gt[e]);
        tb[G_W + t] = dt[e] * ex2_ftz(rest[e]);
        tb[G_EG + t] = t >= fb ? __int_as_float(0x7fc00000) : ex2_ftz(gt[e]);
      }
      if (lane == 0) decs[(c % kGateBufs) * 2 + gh] = fb < 64 ? __int_as_float(0x7fc00000) : ex2_ftz(g63);
    };

    if (gate_warp) {
      prefetch_gates(0);
      compute_gates(0);
      if (n > 1) {
        prefetch_gates(1);
        compute_gates(1);
      }
      if (n > 2) prefetch_gates(2);
    }

    // ---- initial state ------------------------------------------------------
    float s[kCols];
    float dprod = 1.f;  // decay of the piece
    if (!STATE_ONLY && p.state && row_live) {
#pragma unroll
      for (int i = 0; i < kCols / 4; ++i) {
        const float4 v = ld_stream_f4(p.state + row_off + 4 * i);
        s[4 * i] = v.x;
        s[4 * i + 1] = v.y;
        s[4 * i + 2] = v.z;
        s[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCols; ++i) s[i] = 0.f;
    }
    if (!STATE_ONLY) {
      for (int j = 0; j < pc.index; ++j) {  // through the pieces before this one
        const int64_t u = (slot - pc.index + j) * p.tiles + tile;
        const float dec = p.ws_dec[2 * u + hh];
        const float4* F = reinterpret_cast<const float4*>(p.ws) + u * (kRows * NS / 4) + tid;
#pragma unroll
        for (int i = 0; i < kCols / 4; ++i) {
          const float4 v = __ldg(F + i * kComputeThreads);
          s[4 * i] = fmaf(dec, s[4 * i], v.x);
          s[4 * i + 1] = fmaf(dec, s[4 * i + 1], v.y);
          s[4 * i + 2] = fmaf(dec, s[4 * i + 2], v.z);
          s[4 * i + 3] = fmaf(dec, s[4 * i + 3], v.w);
        }
      }
    }
    auto publish_state = [&]() {  // S as the bf16 A operand of (C S)^T
      uint32_t w[kCols / 2];
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) w[i] = pack_bf16x2(s[2 * i], s[2 * i + 1]);
      if constexpr (kCols == 32)
        tmem_st16u(tl + TM_SB + 16 * cq, w);
      else
        tmem_st8u(tl + TM_SB + 8 * cq, w);
      tmem_wait_st();
      signal(B_RDY_S, false);
    };
    if (!STATE_ONLY) publish_state();

    // ---- W of chunk c ---------------------------------------------------------
    const int wtid = STATE_ONLY ? tid : (warp >> 2) * 64 + (warp & 1) * 32 + lane;  // among the W warps
    auto make_w = [&](int c) {
      const uint32_t xs = sb + L::OFF_ST + (c % kStages) * L::kStage;
      wait(B_FULL + c % kStages, static_cast<uint32_t>((c / kStages) & 1));
      if (c > 0) wait(B_DS + ((c - 1) & 1), static_cast<uint32_t>(((c - 1) >> 1) & 1));  // W is free
      const int Lc = static_cast<int>(min(static_cast<int64_t>(kChunk), Ltot - static_cast<int64_t>(c) * kChunk));
      constexpr int kUnits = 1024 / (32 * kWWarps);
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const int idx = wtid + 32 * kWWarps * k;
        const int t = idx >> 4, blk = (idx >> 3) & 1;
        const uint32_t off = blk * 8192 + sw128_off(t, idx & 7);
        uint4 x = lds128(xs + off);
        if (t >= Lc) {  // past the end: x and B of the last chunk become zero
          x = make_uint4(0, 0, 0, 0);
          sts128(xs + off, 0u, 0u, 0u, 0u);
          if (blk < kKb) sts128(xs + L::kX + blk * 16384 + sw128_off(t, idx & 7), 0u, 0u, 0u, 0u);
        }
        const float w = table(c, kHeads == 2 ? blk : 0)[G_W + t];
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
        uint32_t hi[4], lo[4];
        float2 chk = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = __fmul2_rn(make_float2(bf16_lo(xw[e]), bf16_hi(xw[e])), make_float2(w, w));
          hi[e] = pack_bf16x2(v.x, v.y);
          const float2 r = __fadd2_rn(v, make_float2(-bf16_lo(hi[e]), -bf16_hi(hi[e])));
          lo[e] = pack_bf16x2(r.x, r.y);
          chk = __ffma2_rn(r, make_float2(0.f, 0.f), chk);  // NaN where x is not finite
        }
        sts128(sb + L::OFF_W + off, hi[0], hi[1], hi[2], hi[3]);
        sts128(sb + L::OFF_W + 16384 + off, lo[0], lo[1], lo[2], lo[3]);
        if (!STATE_ONLY && !(chk.x + chk.y == 0.f)) {
          uint32_t cl[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            cl[e] = xw[e];
#pragma unroll
            for (int f = 0; f < 2; ++f)
              if (((xw[e] >> (16 * f)) & 0x7f80u) == 0x7f80u) {
                cl[e] &= f ? 0x0000ffffu : 0xffff0000u;
                atomicMin(&first_bad[blk * 64 + 8 * (idx & 7) + 2 * e + f], c * kChunk + t);
                *any_bad = 1u;
              }
          }
          sts128(xs + off, cl[0], cl[1], cl[2], cl[3]);
        }
      }
      signal(B_RDY_W, true);
    };

    // ---- M of chunk c (quarters 2-3: rows i = row - 64, columns [16 cq, 16 cq + 16)) ----
    auto make_m = [&](int c) {
      const uint32_t par = static_cast<uint32_t>(c & 1);
      if (quarter == 2 && cq >= 2) {  // above the diagonal: zero since the start
        signal(B_RDY_M, false);
        return;
      }
      const int i = row - 64, r0 = 16 * cq;
      wait(B_G, par);
      float v[16];
      tmem_ld16(tl + TM_G + r0, v);
      tmem_wait_ld();
      reg_fence(v);
      if (c > 0) wait(B_PV, par ^ 1u);  // M is free
#pragma unroll
      for (int head = 0; head < kHeads; ++head) {
        const float* tb = table(c, head);
        float m[16];
        if (quarter == 3 && cq < 2) {  // below the diagonal
          const float r = ex2_ftz(tb[G_GAM + i] - tb[G_GAM + r0 + 15]);
          float u[16];
          load16(tb + G_U + r0, u);
#pragma unroll
          for (int jj = 0; jj < 16; jj += 2) {
            const float2 q = __fmul2_rn(__fmul2_rn(make_float2(v[jj], v[jj + 1]), make_float2(u[jj], u[jj + 1])),
                                        make_float2(r, r));
            m[jj] = q.x;
            m[jj + 1] = q.y;
          }
        } else {
          const float gi = tb[G_GAM + i];
          const float skip = p.D && (head == 0 || two) ? p.D[h0 + head] : 0.f;
          float dd[16], dt[16];
          load16(tb + G_D + r0, dd);
          load16(tb + G_DT + r0, dt);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int topc = r0 + 4 * q + 3;
            float e = topc <= i ? ex2_ftz(gi - tb[G_GAM + topc]) : 1.f;
#pragma unroll
            for (int jj = 4 * q + 3; jj >= 4 * q; --jj) {
              const int j = r0 + jj;
              m[jj] = j <= i ? fmaf(v[jj], e * dt[jj], j == i ? skip : 0.f) : 0.f;
              e = j > i ? 1.f : e * dd[jj];
            }
          }
        }
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2)
          sts128(sb + L::OFF_M + head * 8192 + sw128_off(i, 2 * cq + c2), pack_bf16x2(m[8 * c2], m[8 * c2 + 1]),
                 pack_bf16x2(m[8 * c2 + 2], m[8 * c2 + 3]), pack_bf16x2(m[8 * c2 + 4], m[8 * c2 + 5]),
                 pack_bf16x2(m[8 * c2 + 6], m[8 * c2 + 7]));
      }
      signal(B_RDY_M, true);
    };

    // ---- outputs of chunk c (row, tokens [16 cq, 16 cq + 16)) -------------------
    auto outputs = [&](int c) {
      const uint32_t par = static_cast<uint32_t>(c & 1);
      const int Lc = static_cast<int>(min(static_cast<int64_t>(kChunk), Ltot - static_cast<int64_t>(c) * kChunk));
      float eg[16], qs[16], pv[16];
      load16(table(c, hh) + G_EG + 16 * cq, eg);
      wait(B_PV, par);
      tmem_ld16(tl + TM_PV + 16 * cq, pv);
      wait(B_QS, par);
      tmem_ld16(tl + TM_QS + 16 * cq, qs);
      tmem_wait_ld();
      reg_fence(pv);
      reg_fence(qs);
      float o[16];
#pragma unroll
      for (int k = 0; k < 16; k += 2) {
        const float2 r = __ffma2_rn(make_float2(eg[k], eg[k + 1]), make_float2(qs[k], qs[k + 1]),
                                    make_float2(pv[k], pv[k + 1]));
        o[k] = r.x;
        o[k + 1] = r.y;
      }
      if (*any_bad) {
        const int fb = first_bad[row] - c * kChunk - 16 * cq;
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (k >= fb) o[k] = __int_as_float(0x7fc00000);
      }
      if (Lc == kChunk) {
        // lanes pair up (row even, row + 1): the even lane stores the bf16x2 words of the first
        // eight tokens, the odd lane those of the rest
        const bool odd = row & 1;
        const uint32_t ocol = sb + L::OFF_Y + (row >> 6) * 8192 + 4 * ((row & 7) >> 1);
        const int och = (row & 63) >> 3;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float mine = odd ? o[8 + k] : o[k];
          const float theirs = __shfl_xor_sync(0xffffffffu, odd ? o[k] : o[8 + k], 1);
          const int t = 16 * cq + (odd ? 8 : 0) + k;
          sts32(ocol + t * 128 + ((och ^ (t & 7)) << 4), odd ? pack_bf16x2(theirs, mine) : pack_bf16x2(mine, theirs));
        }
      } else if (row_live) {
        __nv_bfloat16* dst = p.out + ((bos + static_cast<int64_t>(c) * kChunk + 16 * cq) * p.H + h0 + hh) * P + (row & (P - 1));
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (16 * cq + k < Lc) dst[static_cast<int64_t>(k) * p.H * P] = __float2bfloat16_rn(o[k]);
      }
      signal(B_RDY_D, true);
    };

    // ---- state update of chunk c ------------------------------------------------
    auto update = [&](int c) {
      const float dec = decs[(c % kGateBufs) * 2 + hh];
      dprod *= dec;
      wait(B_DS + (c & 1), static_cast<uint32_t>((c >> 1) & 1));
      float v[kCols];
      if constexpr (kCols == 32)
        tmem_ld32(tl + TM_DS + 128 * (c & 1) + 32 * cq, v);
      else
        tmem_ld16(tl + TM_DS + 128 * (c & 1) + 16 * cq, v);
      tmem_wait_ld();
      reg_fence(v);
#pragma unroll
      for (int i = 0; i < kCols; i += 2) {
        const float2 r = __ffma2_rn(make_float2(dec, dec), make_float2(s[i], s[i + 1]), make_float2(v[i], v[i + 1]));
        s[i] = r.x;
        s[i + 1] = r.y;
      }
      if (!STATE_ONLY && c + 1 < n) publish_state();
    };

    bool aborted = false;
    for (int c = -1; c < n; ++c) {
      tc_fence_before();
      if (failed) *abort_flag = 1u;
      named_sync(kComputeBar, kComputeThreads);  // tables of chunk c + 1; everyone is past chunk c - 1
      tc_fence_after();
      if (*abort_flag) {
        aborted = true;
        break;
      }
      if (c + 1 < n) {
        if (STATE_ONLY || quarter < 2) make_w(c + 1);
        if (!STATE_ONLY && quarter >= 2) make_m(c + 1);
      }
      if (gate_warp && c >= 0 && c + 2 < n) {
        compute_gates(c + 2);
        if (c + 3 < n) prefetch_gates(c + 3);
      }
      if (c >= 0) {
        if (!STATE_ONLY) outputs(c);
        update(c);
      }
    }

    if (!aborted && !failed) {
      if (STATE_ONLY) {
        const int64_t u = slot * p.tiles + tile;
        float4* F = reinterpret_cast<float4*>(p.ws) + u * (kRows * NS / 4) + tid;
#pragma unroll
        for (int i = 0; i < kCols / 4; ++i)
          F[i * kComputeThreads] = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
        if (cq == 0 && (row & 63) == 0) p.ws_dec[2 * u + (row >> 6)] = dprod;
      } else if (last_piece && row_live) {
#pragma unroll
        for (int i = 0; i < kCols / 4; ++i)
          st_stream_f4(p.new_state + row_off + 4 * i, make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]));
      }
    }
  } else if (warp == kMmaWarp) {
    if (lane == 0) {
      // ======================= MMA issue thread ================================
      constexpr uint32_t idesc_g = idesc_bf16(128, 64, false, false);   // [B; C] B^T
      constexpr uint32_t idesc_ds = idesc_bf16(128, NS, true, true);    // W^T B
      constexpr uint32_t idesc_qs = idesc_bf16(128, 64, false, false);  // S (TMEM) C^T
      constexpr uint32_t idesc_pv = idesc_bf16(128, 64, true, false);   // X^T M^T
      const uint32_t sb16 = sb >> 4;
      auto bc16 = [&](int c) { return sb16 + (L::OFF_ST + (c % kStages) * L::kStage + L::kX) / 16; };
      auto wait = [&](int b, uint32_t parity) -> bool {
        if (!mbar_wait(&bars[b], parity, kTimeoutNs)) return false;
        tc_fence_after();
        return true;
      };
      auto mma_g = [&](int c) -> bool {
        if (!wait(B_FULL + c % kStages, static_cast<uint32_t>((c / kStages) & 1))) return false;
#pragma unroll
        for (int ks = 0; ks < NS / 16; ++ks) {
          const uint64_t d = sdesc_sw128_f(bc16(c) + ((ks >> 2) * 16384 + (ks & 3) * 32) / 16, 16, 1024);
          mma_bf16_ss(tmem + TM_G, d, d, idesc_g, ks > 0);
        }
        mma_commit(&bars[B_G]);
        return true;
      };
      auto mma_ds = [&](int c) {
        const uint32_t d = tmem + TM_DS + 128 * (c & 1);
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            mma_bf16_ss(d, sdesc_sw128_f(sb16 + (L::OFF_W + part * 16384 + ks * 2048) / 16, 8192, 1024),
                        sdesc_sw128_f(bc16(c) + ks * 128, 16384, 1024), idesc_ds, part > 0 || ks > 0);
        mma_commit(&bars[B_DS + (c & 1)]);
      };
      auto mma_pv = [&](int c) {
        const uint32_t xo = L::OFF_ST + (c % kStages) * L::kStage;
#pragma unroll
        for (int head = 0; head < kHeads; ++head)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint64_t b = sdesc_sw128_f(sb16 + (L::OFF_M + head * 8192 + ks * 32) / 16, 16, 1024);
            // rows 0-63 and 64-127 of X^T are two blocks of 64; with two heads, the block of the
            // other head is 2 KiB of zeros, so that each head's M meets its own x only
            uint32_t start = xo + ks * 2048, lbo = 8192;
            if (kHeads == 2 && head == 0) lbo = L::OFF_Z1 - start;
            if (kHeads == 2 && head == 1) {
              lbo = start + 8192 - L::OFF_Z0;
              start = L::OFF_Z0;
            }
            mma_bf16_ss(tmem + TM_PV, sdesc_sw128_f(sb16 + start / 16, lbo, 1024), b, idesc_pv, head > 0 || ks > 0);
          }
      };
      auto mma_qs = [&](int c) {
#pragma unroll
        for (int ks = 0; ks < NS / 16; ++ks)
          mma_bf16_ts(tmem + TM_QS, tmem + TM_SB + 8 * ks,
                      sdesc_sw128_f(bc16(c) + ((ks >> 2) * 16384 + 8192 + (ks & 3) * 32) / 16, 16, 1024), idesc_qs, ks > 0);
      };
      bool ok = STATE_ONLY || mma_g(0);
      for (int c = -1; ok && c < n; ++c) {
        const uint32_t next = static_cast<uint32_t>((c + 1) & 1);
        if (c + 1 < n) {
          if (!(ok = wait(B_RDY_W, next))) break;
          mma_ds(c + 1);
          if (STATE_ONLY) {
            mma_commit(&bars[B_EMPTY + (c + 1) % kStages]);
          } else {
            if (!(ok = wait(B_RDY_M, next))) break;
            if (c + 2 < n && !(ok = mma_g(c + 2))) break;
          }
        }
        if (STATE_ONLY) continue;
        if (c >= 0 && !(ok = wait(B_RDY_D, next ^ 1u))) break;  // the outputs of chunk c left their accumulators
        if (c + 1 < n) {
          mma_pv(c + 1);
          mma_commit(&bars[B_PV]);
        }
        if (c >= 0 && Ltot - static_cast<int64_t>(c) * kChunk >= kChunk) {
          const int tok = static_cast<int>(bos + static_cast<int64_t>(c) * kChunk);
          tma_store_3d(&tm_y, smem + L::OFF_Y, 0, h0, tok);
          if (P == 128)
            tma_store_3d(&tm_y, smem + L::OFF_Y + 8192, 64, h0, tok);
          else if (two)
            tma_store_3d(&tm_y, smem + L::OFF_Y + 8192, 0, h0 + 1, tok);
          bulk_commit();
        }
        if (c + 1 < n) {
          if (!(ok = wait(B_RDY_S, next))) break;
          mma_qs(c + 1);
          bulk_wait_read_all();  // the output tile may be written again once B_QS completes
          mma_commit(&bars[B_QS]);
          mma_commit(&bars[B_EMPTY + (c + 1) % kStages]);
        }
      }
      bulk_wait_all();
      mma_commit(&bars[B_END]);
      if (!mbar_wait(&bars[B_END], 0, kTimeoutNs)) ok = false;
      failed = !ok;
    }
  } else if (lane == 0) {
    // ======================= TMA load thread ===================================
    const uint32_t bytes = (kHeads == 2 && !two ? 8192u : 16384u) + kKb * (STATE_ONLY ? 8192u : 16384u);
    bool ok = true;
    int issued = 0;
    for (int c = 0; ok && c < n; ++c) {
      const int st = c % kStages;
      if (c >= kStages && !mbar_wait(&bars[B_EMPTY + st], static_cast<uint32_t>((c / kStages - 1) & 1), kTimeoutNs)) {
        ok = false;
        break;
      }
      const int tok = static_cast<int>(bos + static_cast<int64_t>(c) * kChunk);
      uint64_t* bar = &bars[B_FULL + st];
      uint8_t* xs = smem + L::OFF_ST + st * L::kStage;
      mbar_arrive_expect_tx(bar, bytes);
      if (P == 128) {
        tma_load_3d(xs, &tm_x, bar, 0, h0, tok);
        tma_load_3d(xs + 8192, &tm_x, bar, 64, h0, tok);
      } else {
        tma_load_3d(xs, &tm_x, bar, 0, h0, tok);
        if (two) tma_load_3d(xs + 8192, &tm_x, bar, 0, h0 + 1, tok);
      }
#pragma unroll
      for (int kb = 0; kb < kKb; ++kb) {
        tma_load_3d(xs + L::kX + kb * 16384, &tm_b, bar, 64 * kb, g, tok);
        if (!STATE_ONLY) tma_load_3d(xs + L::kX + kb * 16384 + 8192, &tm_c, bar, 64 * kb, g, tok);
      }
      issued = c + 1;
    }
    // no load may be in flight when the CTA ends
    for (int c = max(0, issued - kStages); c < issued; ++c)
      if (!mbar_wait(&bars[B_FULL + c % kStages], static_cast<uint32_t>((c / kStages) & 1), kTimeoutNs)) ok = false;
    failed = !ok;
  }
  if (failed) atomicOr(&g_ssm_status, kStatusSsmTimeout);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---- host side ---------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

// [T, heads, inner] bf16, box = 64 tokens x 1 head x 64 values, 128-byte swizzle; a small
// cache per thread spares a caller that reuses its buffers the ~1 us of an encoding.
cudaError_t make_map(CUtensorMap* m, const void* base, int64_t inner, int64_t heads, int64_t T) {
  struct Entry {
    const void* base;
    int64_t inner, heads, T;
    CUtensorMap map;
  };
  constexpr int kEntries = 16;
  thread_local Entry cache[kEntries];
  thread_local int used = 0, next = 0;
  for (int i = 0; i < used; ++i)
    if (cache[i].base == base && cache[i].inner == inner && cache[i].heads == heads && cache[i].T == T) {
      *m = cache[i].map;
      return cudaSuccess;
    }
  auto fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(T)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(inner) * 2, static_cast<cuuint64_t>(heads) * inner * 2};
  cuuint32_t box[3] = {64, 1, 64};
  cuuint32_t es[3] = {1, 1, 1};
  if (fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  cache[next] = Entry{base, inner, heads, T, *m};
  next = (next + 1) % kEntries;
  if (used < kEntries) ++used;
  return cudaSuccess;
}

int64_t head_tiles(int64_t H, int64_t G, int64_t P) { return G * ((H / G * P + kRows - 1) / kRows); }

struct Cut {
  int64_t seg = 0;    // tokens of a piece, 0: no cut
  int64_t slots = 0;  // at most so many pieces
};

Cut choose_cut(int64_t T, int64_t N, int64_t tiles, int sms) {
  (void)sms, (void)tiles, (void)T;
  return Cut{0, N};
}

template <int P, int NS, bool STATE_ONLY>
cudaError_t launch_one(const CUtensorMap* m, const Params& p, int64_t slots, cudaStream_t s) {
  auto kernel = gdn_ssm_chunked_kernel<P, NS, STATE_ONLY>;
  constexpr int bytes = Lay<P, NS>::kBytes;
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess) return e;
  const int64_t ctas = slots * p.tiles;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  kernel<<<static_cast<unsigned>(ctas), kThreads, bytes, s>>>(m[0], m[1], m[2], m[3], p);
  return cudaGetLastError();
}

template <int P, int NS>
cudaError_t launch(const SsmArgs& a, const Cut& cut, void* ws, cudaStream_t s) {
  CUtensorMap m[4];
  cudaError_t e;
  if ((e = make_map(&m[0], a.x, P, a.H, a.T)) != cudaSuccess) return e;
  if ((e = make_map(&m[1], a.B, NS, a.G, a.T)) != cudaSuccess) return e;
  if ((e = make_map(&m[2], a.C, NS, a.G, a.T)) != cudaSuccess) return e;
  if ((e = make_map(&m[3], a.out, P, a.H, a.T)) != cudaSuccess) return e;
  Params p{a.state, a.A_log, a.dt_bias, a.D, static_cast<const __nv_bfloat16*>(a.a), a.cu_seqlens,
           static_cast<__nv_bfloat16*>(a.out), a.new_state, static_cast<float*>(ws), nullptr, a.T, a.N, cut.seg,
           static_cast<int>(a.H), static_cast<int>(a.G), static_cast<int>(head_tiles(a.H, a.G, P))};
  if (cut.seg) {
    p.ws_dec = p.ws + cut.slots * p.tiles * kRows * NS;
    if ((e = launch_one<P, NS, true>(m, p, cut.slots, s)) != cudaSuccess) return e;
  }
  return launch_one<P, NS, false>(m, p, cut.slots, s);
}

}  // namespace

size_t ssm_chunked_workspace(int64_t T, int64_t N, int64_t H, int64_t G, int64_t P, int64_t Ns, int sms) {
  const int64_t tiles = head_tiles(H, G, P);
  const Cut cut = choose_cut(T, N, tiles, sms);
  return cut.seg ? static_cast<size_t>(cut.slots) * tiles * (kRows * Ns + 2) * sizeof(float) : 0;
}

cudaError_t launch_ssm_chunked(const SsmArgs& a, void* ws, int sms, cudaStream_t s) {
  const Cut cut = ws ? choose_cut(a.T, a.N, head_tiles(a.H, a.G, a.P), sms) : Cut{0, a.N};
  if (a.P == 64) return a.Ns == 64 ? launch<64, 64>(a, cut, ws, s) : launch<64, 128>(a, cut, ws, s);
  return a.Ns == 64 ? launch<128, 64>(a, cut, ws, s) : launch<128, 128>(a, cut, ws, s);
}

cudaError_t read_ssm_status(uint32_t* out, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_ssm_status, sizeof(uint32_t));
  if (e != cudaSuccess || !clear) return e;
  const uint32_t zero = 0;
  return cudaMemcpyToSymbol(g_ssm_status, &zero, sizeof(uint32_t));
}

}  // namespace gdn
