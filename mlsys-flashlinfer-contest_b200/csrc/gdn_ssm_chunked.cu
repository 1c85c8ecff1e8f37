// Selective state-space scan of packed prompts in chunks of 64 tokens on tcgen05 tensor
// cores (sm_100a).
//
// A CTA owns 128 state rows of one sequence piece: two heads of 64 or one of 128, of one
// B/C group.  With gamma the inclusive cumulative log decay within the chunk and S [128, Ns]
// the state at its start, every accumulator is transposed (a TMEM lane is a state row
// (head, p)):
//   G      = C B^T                                  [i, j]    (one product for all heads)
//   M_h    = G e^{gamma_i - gamma_j} dt_j + D [i = j]  for j <= i
//   (M X)^T = X^T M^T,  (C S)^T = S C^T             [row, i]
//   y^T    = e^{gamma_i} (C S)^T + (M X)^T
//   S     <- e^{gamma_63} S + W^T B,   W = e^{gamma_63 - gamma_j} dt_j x_j
// Roundings: M and the S that C reads are operands of two bf16 terms, the rounded value and what it
// left (16 bits: 2^-16 of a term, where the output's own rounding is 2^-8; with one term each the
// outputs' error was 1.4 times that of their rounding, and the skip factor itself was rounded).  The state
// itself stays fp32 in registers for the whole piece, and W enters its update as three bf16 terms (24
// bits of mantissa; B is bf16 already): the final state is as exact as fp32 sums make it.  Two terms left
// 2.6e-6 of it.  The second terms cost about a tenth of the time (four prompts of 8192 tokens, 64 heads of
// 64: 330 -> 365 us).
//
// The decays between a row and the columns of a 16-column block are r_i u_j.  Below the
// diagonal u_j = dt_j e^{gamma_top - gamma_j} (a table, top = the block's last column) and
// r_i = e^{gamma_i - gamma_top}: no factor exceeds 1, whatever the decay.  In the blocks on the
// diagonal both refer to the block's first column instead, which u_j may exceed by the
// block's decay; where that is more than 2^64 (a flag of the tables), each element gets its own
// exponential.  The mask and the skip term D of a row come from tables in shared memory (a mask
// word per two columns, applied to the packed bf16 values, so that it also hides a NaN).
//
// Two heads of a tile: M X is one product of N = 128, [M_0 | M_1] against the x of both, of which each
// row reads its own head's 64 columns.  Half of it is thrown away, as it would be with a product of
// zeros for each head, but no head's M meets the other's x: what is not finite in one (D, an
// overflow) stays there, and it is half as many MMAs to issue.
//
// Values that are not finite stay where the recurrence puts them.  A masked factor 0 times
// an infinite x would leak into earlier tokens: x that is not finite is replaced by 0 as an operand and
// its row's outputs from that token on are set to NaN; gates that are not finite are 0 in the operands
// and NaN in the decays (e^gamma and the chunk's); tokens past the end are zeroed in x and B.
//
// Warp roles: warps 0-15 compute (four per TMEM lane quarter, each on a quarter of the
// columns), warp 16 issues the MMAs, warp 17 the TMA loads and stores, warps 18-19 compute the
// gate tables of a head each.  The compute warps run, for chunk c: the operands W (quarters
// 0-1) and M (quarters 2-3) of chunk c + 1, the state update of chunk c, the outputs of
// chunk c, which go where the chunk's x was and leave by TMA.  Warps meet through mbarriers only (they
// may be in different steps).  What bounds the kernel is the compute warps' instructions, at five warps a
// scheduler, and the order in which they and the products wait for one another; counted on 16384 tokens, 64
// heads of 64, Ns 128 (195 us): 10900 warp instructions a chunk, issue slots 56 % busy, the tensor pipe 34 %,
// 2200 shared-memory wavefronts a chunk (44 % of the pipe), HBM 20 %.  A chunk of the 4 x 16384 tokens takes 2.7 us
// (692 us); 128 CTAs run there, one an SM, and 20 SMs have none.
//
// Few (sequence, head tile) pairs: sequences are cut into pieces of `seg` tokens.  A first
// launch (STATE_ONLY) finds each piece's final state from zero and its decay; the second runs
// all pieces, each from S = decay S + F over the pieces before it.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "gdn_common.cuh"
#include "gdn_internal.h"
#include "gdn_sm100.cuh"
#include "gdn_tmap.h"

namespace gdn {

__device__ uint32_t g_ssm_status = 0;

namespace {
using namespace sm100;

constexpr int kComputeWarps = 16;
constexpr int kComputeThreads = 32 * kComputeWarps;
constexpr int kMmaWarp = 16, kLoadWarp = 17, kGateWarp = 18;  // and 19: the second head's gates
constexpr int kThreads = kComputeThreads + 128;
constexpr uint32_t kComputeBar = 1;  // named barrier of the compute warps
constexpr uint64_t kTimeoutNs = 2000000000ull;  // 2 s per wait, then give up
constexpr int kStages = 3;
constexpr int kRows = 128;  // state rows of a CTA
constexpr int kTerms = 3;   // bf16 terms of W
constexpr int kMTerms = 2;  // and of M

// ---- TMEM columns ----------------------------------------------------------
constexpr uint32_t TM_G = 0;     // lanes 64-127: G [i][j]
constexpr uint32_t TM_DS = 64;   // W^T B [row][n] (STATE_ONLY: two buffers of 128 columns)
constexpr uint32_t TM_QS = 192;  // (C S)^T [row][i]
constexpr uint32_t TM_PV = 256;  // (M X)^T [row][head of M][i]
constexpr uint32_t TM_SB = 384;  // the two bf16 terms of S [term][row][n]: A operands, 64 columns each
constexpr uint32_t kTmemCols = 512;

// ---- per-token tables (floats) of one head and chunk ------------------------
constexpr int G_GAM = 0;    // gamma, in log2 units
constexpr int G_V = 64;     // dt 2^(gamma of the first token of t's 16 - gamma_t)
constexpr int G_DT = 128;   // dt (0 past the end)
constexpr int G_U = 192;    // dt 2^(gamma of the last token of t's 16 - gamma_t)
constexpr int G_W = 256;    // dt 2^(gamma_63 - gamma_t)
constexpr int G_EG = 320;   // 2^gamma_t
constexpr int G_LOW = 384;  // what gamma's rounding to fp32 left of it
constexpr int kGateFloats = 448;

// ---- shared memory (offsets from a 1024-aligned base) ------------------------
template <int P, int NS>
struct Lay {
  static constexpr int kHeads = kRows / P;   // heads of a tile
  static constexpr int kKb = NS / 64;        // 64-column blocks of B and C
  // B and C of a chunk are done with before its x, whose place its outputs take: two stages are
  // enough for them where three do not fit
  static constexpr int kBcStages = kHeads * kKb > 2 ? 2 : 3;
  static constexpr uint32_t kX = 16384;         // [block 2][t 64][128 B]
  static constexpr uint32_t kBc = kKb * 16384;  // [kb][B 64 rows | C 64 rows][128 B]
  static constexpr uint32_t OFF_X = 0;
  static constexpr uint32_t OFF_BC = OFF_X + kStages * kX;
  static constexpr uint32_t OFF_W = OFF_BC + kBcStages * kBc;  // the terms of W: [term 3][block 2][t 64][128 B]
  static constexpr uint32_t OFF_M = OFF_W + kTerms * 16384;  // the terms of M: [term 2][head][i 64][128 B]
  static constexpr uint32_t kM = kHeads * 8192;
  static constexpr uint32_t OFF_G = OFF_M + (kMTerms * kM < 16384 ? 16384 : kMTerms * kM);  // tables [buffer][head][kGateFloats]
  static constexpr uint32_t OFF_DEC = OFF_G + kStages * 2 * kGateFloats * 4;  // [buffer][head]
  static constexpr uint32_t OFF_STEEP = OFF_DEC + 32;  // [buffer][head]: a bit per 16-block of G_V out of range
  static constexpr uint32_t OFF_BAD = OFF_STEEP + 32;  // first token whose x is not finite, by row
  // by a row's distance from its block's first column, clamped to -1..16 (row 0 is -1): mask
  // words of the 16 columns, and D at the diagonal of each head (pitches free of bank conflicts)
  static constexpr uint32_t OFF_MASK = OFF_BAD + kRows * 4;
  static constexpr uint32_t kMaskPitch = 48, kSkipPitch = 80, kSkipHead = 18 * kSkipPitch;
  static constexpr uint32_t OFF_SKIP = OFF_MASK + 18 * kMaskPitch;
  static constexpr uint32_t OFF_BAR = OFF_SKIP + 2 * kSkipHead;
  static constexpr uint32_t kBytes = OFF_BAR + 256 + 1024;
};
static_assert(Lay<64, 128>::kBytes <= 232448 && Lay<128, 128>::kBytes <= 232448, "shared memory");

enum : int {
  B_BC = 0,                 // kBcStages: a chunk's B and C landed
  B_X = B_BC + kStages,     // kStages: its x landed and its tables are written
  B_EMPTY = B_X + kStages,  // kBcStages: every product that reads its B, C and x is done
  B_DONE = B_EMPTY + kStages,  // kStages: the compute warps are through with a chunk
  B_RDY_W = B_DONE + kStages, B_RDY_M,  // compute warps -> issue warp: operands of a chunk,
  B_RDY_S, B_RDY_D,                     // W^T B of the chunk before read, its other accumulators read
  B_G, B_DS, B_DS1, B_PV, B_QS, B_END,  // products done (two of W^T B with STATE_ONLY: its buffers)
  B_STATE,  // the initial state landed
  kNumBars
};
static_assert(kNumBars * 8 + 8 <= 256, "barrier area");

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
  int64_t inner;    // pieces that are not a sequence's last, at most
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

// Shared-memory store of an operand that only the tensor pipe reads: without a compiler barrier,
// so that loads of tables and the arithmetic of the next piece may pass it.
__device__ __forceinline__ void sts128_op(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d));
}

__device__ __forceinline__ void sts32_op(uint32_t addr, uint32_t a) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(a));
}

// The MMAs are issued from code that the whole warp runs, each instruction by one lane
// (`leader`): descriptors then stay in uniform registers.  In a branch of one lane every
// descriptor is built in vector registers and moved over, ~100 cycles an MMA.
__device__ __forceinline__ void mma_ss_by(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts_by(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit_by(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}
// What two values leave when their bf16 roundings (packed in `hi`) are taken off: x - hi is exact in fp32.
__device__ __forceinline__ float2 minus_bf16x2(float2 x, uint32_t hi) {
  float2 r;
  asm("{\n\t.reg .b16 l, h, m;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "mov.b16 m, 0xBF80;\n\t"
      "fma.rn.f32.bf16 %0, l, m, %3;\n\t"
      "fma.rn.f32.bf16 %1, h, m, %4;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(hi), "f"(x.x), "f"(x.y));
  return r;
}
// One lane of the (converged) warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}

// Programmatic dependent launch: lets the next launch start, and waits for the end of the one
// before (at once when this launch was not made that way).
__device__ __forceinline__ void dependency_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The long form of a wait, out of line: polls with short naps, gives up after kTimeoutNs.
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity) { return mbar_wait_nap(bar, parity, kTimeoutNs); }

struct Piece {
  int64_t seq, bos, eos;  // sequence (-1: none) and the piece's tokens
  int index, count;       // of the sequence's pieces
  int before;             // inner pieces of the sequences before this one (where index > 0)
};

// The pieces of a sequence number max(1, ceil(length / seg)); all but its last are inner pieces,
// numbered through the sequences in order.  Four consecutive sequences of a lane, from n0 on: their
// inner pieces `cnt`, bounds and the sum over this lane and those before it.
struct Inner {
  int b[4], e[4], cnt[4], sum, incl;
};
__device__ __forceinline__ Inner inner_pieces(const Params& p, int64_t n0) {
  const int lane = threadIdx.x & 31;
  const unsigned seg = static_cast<unsigned>(p.seg);
  Inner r;
  int64_t c[5];
#pragma unroll
  for (int u = 0; u < 5; ++u) c[u] = p.cu[min(n0 + u, p.N)];
  r.sum = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    r.b[u] = static_cast<int>(min(max(c[u], int64_t(0)), p.T));
    r.e[u] = static_cast<int>(min(max(c[u + 1], static_cast<int64_t>(r.b[u])), p.T));
    const unsigned len = static_cast<unsigned>(r.e[u] - r.b[u]);
    r.cnt[u] = n0 + u < p.N && len > seg ? static_cast<int>((len + seg - 1) / seg) - 1 : 0;
    r.sum += r.cnt[u];
  }
  r.incl = r.sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, r.incl, d);
    if (lane >= d) r.incl += y;
  }
  return r;
}

// The piece of slot `slot`: inner pieces first (the longest run first), then the sequences' last
// ones, whose sequence is the slot itself.  A warp finds an inner piece by itself, 128 sequences
// at a time, and so what lies before a last piece that is not the only one; were all pieces in the
// sequences' order, every CTA would search: 4096 sequences of 64 tokens took 4.6 ms instead of 1.7.
template <bool STATE_ONLY>
__device__ __forceinline__ Piece find_piece(const Params& p, int64_t slot) {
  const int lane = threadIdx.x & 31;
  Piece r{-1, 0, 0, 0, 1, 0};
  if (p.seg == 0 || (!STATE_ONLY && slot >= p.inner)) {
    const int64_t seq = p.seg == 0 ? slot : slot - p.inner;
    if (seq >= p.N) return r;
    r.seq = seq;
    r.bos = min(max(p.cu[seq], int64_t(0)), p.T);
    r.eos = min(max(p.cu[seq + 1], r.bos), p.T);
    if (p.seg == 0 || r.eos - r.bos <= p.seg) return r;
    r.count = static_cast<int>((r.eos - r.bos + p.seg - 1) / p.seg);
    r.index = r.count - 1;
    r.bos += r.index * p.seg;
    for (int64_t base = 0; base < seq; base += 128) {
      const int64_t n0 = base + 4 * lane;
      const Inner in = inner_pieces(p, n0);
      int sum = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) sum += n0 + u < seq ? in.cnt[u] : 0;
      r.before += __reduce_add_sync(0xffffffffu, sum);
    }
    return r;
  }
  int left = static_cast<int>(slot);  // (slots are fewer than 2^31)
  for (int64_t base = 0; base < p.N; base += 128) {
    const Inner in = inner_pieces(p, base + 4 * lane);
    const unsigned hit = __ballot_sync(0xffffffffu, left < in.incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      int at = left - (in.incl - in.sum), k = 0;  // (lane src: the slot among its four sequences' pieces)
#pragma unroll
      for (int u = 0; u < 3; ++u)
        if (k == u && at >= in.cnt[u]) {
          at -= in.cnt[u];
          k = u + 1;
        }
      int bb = in.b[0], ee = in.e[0], cc = in.cnt[0];
#pragma unroll
      for (int u = 1; u < 4; ++u)
        if (k == u) {
          bb = in.b[u];
          ee = in.e[u];
          cc = in.cnt[u];
        }
      r.seq = base + 4 * src + __shfl_sync(0xffffffffu, k, src);
      r.index = __shfl_sync(0xffffffffu, at, src);
      r.count = __shfl_sync(0xffffffffu, cc, src) + 1;
      r.before = static_cast<int>(slot) - r.index;
      r.bos = __shfl_sync(0xffffffffu, bb, src) + r.index * p.seg;
      r.eos = min(r.bos + p.seg, static_cast<int64_t>(__shfl_sync(0xffffffffu, ee, src)));
      return r;
    }
    left -= __shfl_sync(0xffffffffu, in.incl, 31);
  }
  return r;
}

template <int P, int NS, bool STATE_ONLY>
__global__ void __launch_bounds__(kThreads, 1)
    gdn_ssm_chunked_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_b,
                           const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ CUtensorMap tm_y,
                           const __grid_constant__ CUtensorMap tm_s, const __grid_constant__ CUtensorMap tm_n, const Params p) {
  using L = Lay<P, NS>;
  constexpr int kHeads = L::kHeads, kKb = L::kKb, kBcStages = L::kBcStages;
  constexpr int kCols = NS / 4;  // state columns of a compute thread
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sb = smem_u32(smem);
  float* gates = reinterpret_cast<float*>(smem + L::OFF_G);
  float* decs = reinterpret_cast<float*>(smem + L::OFF_DEC);
  uint32_t* steep = reinterpret_cast<uint32_t*>(smem + L::OFF_STEEP);
  int* first_bad = reinterpret_cast<int*>(smem + L::OFF_BAD);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
  volatile uint32_t* any_bad = tmem_slot + 1;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = static_cast<int>(blockIdx.x % p.tiles);
  const int64_t slot = blockIdx.x / p.tiles;
  const int group_heads = p.H / p.G;
  const int group_tiles = p.tiles / p.G;
  const int g = tile / group_tiles;
  const int h0 = g * group_heads + (tile % group_tiles) * kHeads;  // first head of the tile
  const bool two = kHeads == 2 && h0 + 1 < (g + 1) * group_heads;  // its second head exists

  // The second launch may start once every CTA of the first has (it fills the SMs that the first
  // leaves idle).  Its CTAs wait for the first's end where they need its results, and one before it
  // ends, so that the second does not end first.  (Were that all of them, the first's time would
  // not overlap more than a CTA an SM: 1024 sequences of 32 tokens and one of 32 thousand, 64 heads,
  // 2247 instead of 2572 us.)
  if (STATE_ONLY) dependency_launch();
  const bool ends_last = !STATE_ONLY && blockIdx.x == 0;
  const Piece pc = find_piece<STATE_ONLY>(p, slot);
  if (pc.seq < 0) {
    if (ends_last) dependency_wait();
    return;
  }
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
    if (ends_last) dependency_wait();
    return;
  }

  // ---- set-up.  The load thread makes the barriers and starts its loads at once. --------------
  const uint32_t x_bytes = kHeads == 2 && !two ? 8192u : 16384u;
  int bc_issued = 0, x_issued = 0;  // (load thread)
  auto load_bc = [&](int c) {
    const int st = c % kBcStages, tok = static_cast<int>(bos + static_cast<int64_t>(c) * kChunk);
    uint8_t* bc = smem + L::OFF_BC + st * L::kBc;
    mbar_arrive_expect_tx(&bars[B_BC + st], kKb * (STATE_ONLY ? 8192u : 16384u));
#pragma unroll
    for (int kb = 0; kb < kKb; ++kb) {
      tma_load_3d(bc + kb * 16384, &tm_b, &bars[B_BC + st], 64 * kb, g, tok);
      if (!STATE_ONLY) tma_load_3d(bc + kb * 16384 + 8192, &tm_c, &bars[B_BC + st], 64 * kb, g, tok);
    }
    bc_issued = c + 1;
  };
  auto load_x = [&](int c) {
    const int st = c % kStages, tok = static_cast<int>(bos + static_cast<int64_t>(c) * kChunk);
    uint8_t* xs = smem + L::OFF_X + st * L::kX;
    mbar_arrive_expect_tx(&bars[B_X + st], x_bytes);
    tma_load_3d(xs, &tm_x, &bars[B_X + st], 0, h0, tok);
    if (P == 128)
      tma_load_3d(xs + 8192, &tm_x, &bars[B_X + st], 64, h0, tok);
    else if (two)
      tma_load_3d(xs + 8192, &tm_x, &bars[B_X + st], 0, h0 + 1, tok);
    x_issued = c + 1;
  };
  // The initial and the final state pass through the space of W and M (64 KiB, free before the
  // first chunk's and after the last one's) as boxes of 32 columns and 64 rows in the 128-byte
  // swizzle: a thread's own row, read or written directly, is a transaction a lane.
  const bool state_in = !STATE_ONLY && p.state != nullptr;
  const int state_row = static_cast<int>((pc.seq * p.H + h0) * P);
  if (warp == kLoadWarp && lane == 0) {
    for (int i = 0; i < kNumBars; ++i)
      mbar_init(&bars[i], i == B_RDY_W ? (STATE_ONLY ? kComputeWarps : kComputeWarps / 2) : i == B_RDY_M ? (kHeads == 2 ? 8 : 6)
                         : (i == B_RDY_S || i == B_RDY_D || (i >= B_DONE && i < B_DONE + kStages)) ? kComputeWarps
                         : i >= B_X && i < B_EMPTY ? 1 + kHeads : 1);
    fence_mbar_init();
    *any_bad = 0u;
    if (state_in) {
      mbar_arrive_expect_tx(&bars[B_STATE], NS / 32 * (kHeads == 2 && !two ? 8192u : 16384u));
#pragma unroll
      for (int cb = 0; cb < NS / 32; ++cb) {
        tma_load_2d(smem + L::OFF_W + cb * 16384, &tm_s, &bars[B_STATE], 32 * cb, state_row);
        if (P == 128 || two) tma_load_2d(smem + L::OFF_W + cb * 16384 + 8192, &tm_s, &bars[B_STATE], 32 * cb, state_row + 64);
      }
    }
    for (int c = 0; c < min(n, kStages); ++c) {
      if (c < kBcStages) load_bc(c);
      load_x(c);
    }
    if (!STATE_ONLY) prefetch_tmap(&tm_y);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  if (tid < kRows) first_bad[tid] = 0x7fffffff;
  if (!STATE_ONLY) {
    float skip[2] = {0.f, 0.f};
    if (p.D) {
      skip[0] = p.D[h0];
      if (two) skip[1] = p.D[h0 + 1];
    }
    for (int i = tid; i < 18 * 16; i += kThreads) {
      const int d = i / 16 - 1, j = i % 16;
      reinterpret_cast<uint16_t*>(smem + L::OFF_MASK + (d + 1) * L::kMaskPitch)[j] = j <= d ? 0xffffu : 0u;
      for (int head = 0; head < kHeads; ++head)
        reinterpret_cast<float*>(smem + L::OFF_SKIP + head * L::kSkipHead + (d + 1) * L::kSkipPitch)[j] =
            j == d ? skip[head] : 0.f;
    }
  }
  if (kHeads == 2 && !two)  // the absent head's x
    for (int i = tid; i < kStages * 512; i += kThreads)
      sts128(sb + L::OFF_X + (i >> 9) * L::kX + 8192 + 16 * (i & 511), 0u, 0u, 0u, 0u);
  // (gate warps: head gh, two tokens a lane)
  const int gh = warp - kGateWarp;
  const bool live = warp >= kGateWarp && (gh == 0 || (kHeads == 2 && two));
  const unsigned short* pa = reinterpret_cast<const unsigned short*>(p.a) + h0 + (live ? gh : 0);
  unsigned short raw[2] = {0, 0};
  auto load_gates = [&](int c) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t t = bos + static_cast<int64_t>(c) * kChunk + 2 * lane + e;
      if (live && t < pc.eos) raw[e] = pa[t * p.H];
    }
  };
  float negA = 0.f, bias = 0.f;
  if (live) {
    negA = -expf(p.A_log[h0 + gh]) * kLog2e;
    bias = p.dt_bias[h0 + gh];
    load_gates(0);
  }
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
    // After a timeout a lane waits for nothing any more (its results are garbage, the status word
    // says so), and its warp leaves the loop; the warps that waited for it time out in turn.  A test may
    // answer the lanes differently, and the tensor-memory instructions behind it are the whole warp's: they
    // meet first.  A wait costs ~200 cycles of a chunk's ~4700 even when nothing is left to wait for, so the
    // warps make none that another covers: a commit stands for every product issued before it.  (Six
    // waits a chunk instead of four to five, and a flag for timeouts read every chunk: 2-10 %.)
    auto wait = [&](int b, uint32_t parity) {
      if (!failed && !mbar_test(&bars[b], parity)) failed = !wait_long(&bars[b], parity);
      __syncwarp();
      tc_fence_after();
    };
    auto table = [&](int buf, int head) { return gates + (buf * 2 + head) * kGateFloats; };

    // ---- initial state ------------------------------------------------------
    float s[kCols];
    float dprod = 1.f;  // decay of the piece
    const uint32_t state_smem = sb + L::OFF_W + row * 128;
    if (state_in) {
      wait(B_STATE, 0);
#pragma unroll
      for (int i = 0; i < kCols / 4; ++i) {
        const int col = kCols * cq + 4 * i;
        const uint4 v = lds128(state_smem + (col >> 5) * 16384 + (((col >> 2 & 7) ^ (row & 7)) << 4));
        s[4 * i] = __uint_as_float(v.x);
        s[4 * i + 1] = __uint_as_float(v.y);
        s[4 * i + 2] = __uint_as_float(v.z);
        s[4 * i + 3] = __uint_as_float(v.w);
      }
      if (!row_live) {
#pragma unroll
        for (int i = 0; i < kCols; ++i) s[i] = 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCols; ++i) s[i] = 0.f;
    }
    if (!STATE_ONLY) {  // the blocks of M that no warp writes (rows 0-31, columns 32-63) are zero from here on
      if (state_in) named_sync(kComputeBar, kComputeThreads);  // (every thread has its state)
      for (int i = tid; i < static_cast<int>(kMTerms * kHeads * 128); i += kComputeThreads)
        sts128(sb + L::OFF_M + (i >> 7) * 8192 + sw128_off(i >> 2 & 31, 4 + (i & 3)), 0u, 0u, 0u, 0u);
      fence_async_smem();
      named_sync(kComputeBar, kComputeThreads);
    }
    if (!STATE_ONLY) {
      if (pc.index > 0) dependency_wait();  // the first launch's results
      for (int j = 0; j < pc.index; ++j) {  // through the pieces before this one
        // (the bound holds for any cu_seqlens)
        const int64_t u = min(static_cast<int64_t>(pc.before) + j, p.inner - 1) * p.tiles + tile;
        // (coherent loads, past L1: this grid is resident while the first launch still writes the
        // pieces' states, so the read-only path, which wants memory that nobody writes for the whole life of the
        // grid, may not be taken)
        const float dec = __ldcg(p.ws_dec + 2 * u + hh);
        const float4* F = reinterpret_cast<const float4*>(p.ws) + u * (kRows * NS / 4) + tid;
#pragma unroll
        for (int i = 0; i < kCols / 4; ++i) {
          const float4 v = __ldcg(F + i * kComputeThreads);
          s[4 * i] = fmaf(dec, s[4 * i], v.x);
          s[4 * i + 1] = fmaf(dec, s[4 * i + 1], v.y);
          s[4 * i + 2] = fmaf(dec, s[4 * i + 2], v.z);
          s[4 * i + 3] = fmaf(dec, s[4 * i + 3], v.w);
        }
      }
    }
    // a value as bf16 terms: the rounded value, then what it left
    auto split = [](float2 q, uint32_t& hi, uint32_t& lo) {
      hi = pack_bf16x2(q.x, q.y);
      const float2 r = minus_bf16x2(q, hi);
      lo = pack_bf16x2(r.x, r.y);
    };
    auto publish_state = [&]() {  // S as the A operands of (C S)^T
      const uint32_t dst = tl + TM_SB + kCols / 2 * cq;
#pragma unroll
      for (int part = 0; part < kCols / 16; ++part) {
        uint32_t w[8], wl[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split(make_float2(s[16 * part + 2 * i], s[16 * part + 2 * i + 1]), w[i], wl[i]);
        tmem_st8u(dst + 8 * part, w);
        tmem_st8u(dst + 64 + 8 * part, wl);
      }
      tmem_wait_st();
    };
    if (!STATE_ONLY) {
      publish_state();
      signal(B_RDY_S, false);
    }
    constexpr int kDsBufs = STATE_ONLY ? 2 : 1;
    auto wait_ds = [&](int c) { wait(B_DS + c % kDsBufs, static_cast<uint32_t>((c / kDsBufs) & 1)); };
    auto wait_last = [&](int c) {  // every product of chunk c
      if (STATE_ONLY)
        wait_ds(c);
      else
        wait(B_QS, static_cast<uint32_t>(c & 1));
    };

    // ---- W of chunk c by quarters 0-1, in 16-byte pieces of x: a warp takes two tokens at a
    //      time (a token on 16 lanes), four times, 16 tokens apart.  (STATE_ONLY: every warp, twice,
    //      32 apart.)  Shares of it for quarters 2-3 gained nothing or cost 5-20 %. -----------------
    const bool has_w = STATE_ONLY || quarter < 2;
    const int wt = (STATE_ONLY ? 2 * warp : (warp >> 2) * 4 + (warp & 1) * 2) + (lane >> 4);
    const int wblk = (lane >> 3) & 1;
    const uint32_t woff = wblk * 8192 + sw128_off(wt, lane & 7);
    constexpr int kStride = STATE_ONLY ? 32 : 16, kCount = kChunk / kStride;
    auto make_w = [&](int c, int st, uint32_t st_par) {
      const uint32_t xs = sb + L::OFF_X + st * L::kX + woff;
      const int Lc = static_cast<int>(min(static_cast<int64_t>(kChunk), Ltot - static_cast<int64_t>(c) * kChunk));
      wait(B_X + st, st_par);
      uint4 x[kCount];
      float w[kCount];
#pragma unroll
      for (int k = 0; k < kCount; ++k) {
        x[k] = lds128(xs + k * (kStride * 128));
        w[k] = table(st, kHeads == 2 ? wblk : 0)[G_W + wt + kStride * k];
      }
      if (Lc < kChunk) {  // tokens past the end: x and B become zero
        wait(B_BC + c % kBcStages, static_cast<uint32_t>((c / kBcStages) & 1));
        const uint32_t bs = sb + L::OFF_BC + c % kBcStages * L::kBc + wblk * 8192 + woff;  // (blocks 16 KiB apart)
#pragma unroll
        for (int k = 0; k < kCount; ++k)
          if (wt + kStride * k >= Lc) {
            x[k] = make_uint4(0, 0, 0, 0);
            sts128(xs + k * (kStride * 128), 0u, 0u, 0u, 0u);
            if (wblk < kKb) sts128(bs + k * (kStride * 128), 0u, 0u, 0u, 0u);
          }
      }
      if (c > 0) wait_ds(c - 1);  // W is free
      float2 chk = make_float2(0.f, 0.f);
      float2 v[kCount][4];
#pragma unroll
      for (int k = 0; k < kCount; ++k) {
        const uint32_t xw[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[k][e] = __fmul2_rn(make_float2(bf16_lo(xw[e]), bf16_hi(xw[e])), make_float2(w[k], w[k]));
      }
#pragma unroll
      for (int term = 0; term < kTerms; ++term) {  // the rounded value, then what it left
        uint32_t b[kCount][4];
#pragma unroll
        for (int k = 0; k < kCount; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) b[k][e] = pack_bf16x2(v[k][e].x, v[k][e].y);
#pragma unroll
        for (int k = 0; k < kCount; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (term + 1 < kTerms)  // (a product with -1: packed operands have no sign modifier)
              v[k][e] = minus_bf16x2(v[k][e], b[k][e]);
            else
              chk = __fadd2_rn(chk, v[k][e]);  // the last remainders: NaN where x is not finite
#pragma unroll
        for (int k = 0; k < kCount; ++k)
          sts128_op(sb + L::OFF_W + woff + term * 16384 + k * (kStride * 128), b[k][0], b[k][1], b[k][2], b[k][3]);
      }
      if (!STATE_ONLY && !(chk.x + chk.y == chk.x + chk.y)) {
#pragma unroll 1
        for (int k = 0; k < kCount; ++k) {
          const uint4 xr = lds128(xs + k * (kStride * 128));
          uint32_t xw[4] = {xr.x, xr.y, xr.z, xr.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int f = 0; f < 2; ++f)
              if (((xw[e] >> (16 * f)) & 0x7f80u) == 0x7f80u) {
                xw[e] &= f ? 0x0000ffffu : 0xffff0000u;
                atomicMin(&first_bad[wblk * 64 + 8 * (lane & 7) + 2 * e + f], c * kChunk + wt + kStride * k);
                *any_bad = 1u;
              }
          sts128(xs + k * (kStride * 128), xw[0], xw[1], xw[2], xw[3]);
        }
      }
      signal(B_RDY_W, true);
    };

    // ---- M of chunk c: rows i = row - 64 on quarters 2-3, in blocks of 16 columns.  Below the
    //      diagonal a block costs about half of one on it.  With two heads a warp of quarter 2 takes
    //      one block on the diagonal, a warp of quarter 3 one of each kind of one head; with one head
    //      every block has its own warp (two are zero since the start) -----------------------
    const int mi = row - 64;
    const bool has_m = quarter >= 2 && (kHeads == 2 || quarter == 3 || cq < 2);
    auto m_block = [&](auto below, int cb, int head, int st) {
      constexpr bool kBelow = decltype(below)::value;  // the block lies below the diagonal
      const int r0 = 16 * cb;
      const float* tb = table(st, head);
      const int ref = r0 + (kBelow ? 15 : 0);
      const float r = ex2_ftz((tb[G_GAM + mi] - tb[G_GAM + ref]) + (tb[G_LOW + mi] - tb[G_LOW + ref]));
      const bool far = !kBelow && (steep[st * 2 + head] >> cb & 1u);
      float v[16];
      tmem_ld16(tl + TM_G + r0, v);
      tmem_wait_ld();
      reg_fence(v);
      uint32_t m[8], ml[8];
      if constexpr (kBelow) {
        float u[16];
        load16(tb + G_U + r0, u);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2 q = __fmul2_rn(__fmul2_rn(make_float2(v[2 * k], v[2 * k + 1]), make_float2(u[2 * k], u[2 * k + 1])),
                                      make_float2(r, r));
          split(q, m[k], ml[k]);
        }
      } else {
        const int md = min(max(mi - r0, -1), 16) + 1;  // row of the mask and skip tables
        float2 q[8];
        float u[16], rr = r;
        if (!far) {
          load16(tb + G_V + r0, u);
        } else {
          const float gi = tb[G_GAM + mi], li = tb[G_LOW + mi];
          rr = 1.f;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int j = r0 + k;
            u[k] = ex2_ftz(fminf((gi - tb[G_GAM + j]) + (li - tb[G_LOW + j]), 0.f)) * tb[G_DT + j];
          }
        }
        float skip[16];
        load16(reinterpret_cast<const float*>(smem + L::OFF_SKIP + head * L::kSkipHead + md * L::kSkipPitch), skip);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          q[k] = __ffma2_rn(__fmul2_rn(make_float2(v[2 * k], v[2 * k + 1]), make_float2(u[2 * k], u[2 * k + 1])),
                            make_float2(rr, rr), make_float2(skip[2 * k], skip[2 * k + 1]));
        const uint4* mask = reinterpret_cast<const uint4*>(smem + L::OFF_MASK + md * L::kMaskPitch);
#pragma unroll
        for (int k4 = 0; k4 < 2; ++k4) {
          const uint4 a = mask[k4];
          const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            split(q[4 * k4 + k], m[4 * k4 + k], ml[4 * k4 + k]);
            m[4 * k4 + k] &= aw[k];
            ml[4 * k4 + k] &= aw[k];
          }
        }
      }
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        const uint32_t dst = sb + L::OFF_M + head * 8192 + sw128_off(mi, 2 * cb + c2);
        sts128_op(dst, m[4 * c2], m[4 * c2 + 1], m[4 * c2 + 2], m[4 * c2 + 3]);
        sts128_op(dst + L::kM, ml[4 * c2], ml[4 * c2 + 1], ml[4 * c2 + 2], ml[4 * c2 + 3]);
      }
    };
    auto make_m = [&](int c, int st, uint32_t st_par) {
      wait(B_X + st, st_par);  // (the tables)
      // M is free, and G of this chunk, issued before, is there (a commit covers all products before it)
      if (c > 0)
        wait(B_PV, static_cast<uint32_t>((c - 1) & 1));
      else
        wait(B_G, 0);
      if (kHeads == 2) {
        if (quarter == 2) {
          m_block(std::false_type{}, cq & 1, cq >> 1, st);
        } else {
          m_block(std::false_type{}, 2 + (cq >> 1), cq & 1, st);
          m_block(std::true_type{}, cq >> 1, cq & 1, st);
        }
      } else if (quarter == 3 && cq < 2) {
        m_block(std::true_type{}, cq, 0, st);
      } else {
        m_block(std::false_type{}, cq, 0, st);
      }
      signal(B_RDY_M, true);
    };

    // ---- outputs of chunk c (row, tokens [16 cq, 16 cq + 16)).  Lanes pair up (row even,
    //      row + 1) to form bf16x2 words of two rows: at step k the even lane gets token k's, the
    //      odd lane token 8 + (k ^ 4)'s (the other half of a 128-byte line in the swizzle: no
    //      bank is met twice).  They go where the chunk's x was, and from there by TMA ----
    const bool odd = row & 1;
    const uint32_t pick = odd ? 0x3276u : 0x5410u;
    const uint32_t ysm = (row >> 6) * 8192 + (16 * cq + (odd ? 8 : 0)) * 128 + 4 * ((row & 7) >> 1);
    const uint32_t ych = (row & 63) >> 3;
    auto outputs = [&](int c, int st) {
      float eg[16], qs[16], pv[16];
      load16(table(st, hh) + G_EG + 16 * cq, eg);
      const bool bad = *any_bad != 0u;  // (written before this chunk's W was signalled)
      tmem_ld16(tl + TM_PV + 64 * hh + 16 * cq, pv);
      tmem_ld16(tl + TM_QS + 16 * cq, qs);
      tmem_wait_ld();
      reg_fence(pv);
      reg_fence(qs);
      signal(B_RDY_D, false);
      float o[16];
#pragma unroll
      for (int k = 0; k < 16; k += 2) {
        const float2 r = __ffma2_rn(make_float2(eg[k], eg[k + 1]), make_float2(qs[k], qs[k + 1]),
                                    make_float2(pv[k], pv[k + 1]));
        o[k] = r.x;
        o[k + 1] = r.y;
      }
      if (bad) {
        const int fb = first_bad[row] - c * kChunk - 16 * cq;
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (k >= fb) o[k] = __int_as_float(0x7fc00000);
      }
      uint32_t w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t mine = pack_bf16x2(o[k], o[8 + (k ^ 4)]);
        w[k] = __byte_perm(mine, __shfl_xor_sync(0xffffffffu, mine, 1), pick);
      }
      const int64_t left = Ltot - static_cast<int64_t>(c) * kChunk;
      if (!row_live) return;
      if (left >= kChunk) {
        const uint32_t ys = sb + L::OFF_X + st * L::kX + ysm;
#pragma unroll
        for (int k = 0; k < 8; ++k) {  // token k or k ^ 4 of eight: its row, and its swizzle
          const uint32_t t = odd ? k ^ 4 : k;
          sts32_op(ys + t * 128 + ((ych ^ t) << 4), w[k]);
        }
      } else {
        __nv_bfloat16* dst = p.out + ((bos + static_cast<int64_t>(c) * kChunk + 16 * cq + (odd ? 8 : 0)) * p.H + h0 + hh) * P +
                             (row & (P - 2));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int t = odd ? k ^ 4 : k;
          if (16 * cq + (odd ? 8 : 0) + t < left)
            *reinterpret_cast<uint32_t*>(dst + static_cast<int64_t>(t) * p.H * P) = w[k];
        }
      }
    };

    // ---- state update of chunk c ------------------------------------------------
    auto update = [&](int c, int st) {
      const float dec = decs[st * 2 + hh];
      dprod *= dec;
      // W^T B is there: the warps that wrote W or M of the next chunk waited for it, or for M X, which comes
      // after it; the others wait for C S, the chunk's last product
      const bool met = c + 1 < n && (has_w || has_m);
      if (!met) wait_last(c);
      float v[kCols];
      if constexpr (kCols == 32)
        tmem_ld32(tl + TM_DS + 128 * (c % kDsBufs) + 32 * cq, v);
      else
        tmem_ld16(tl + TM_DS + 128 * (c % kDsBufs) + 16 * cq, v);
      tmem_wait_ld();
      reg_fence(v);
      // W^T B has been read: the next may be formed.  (With heads of 64, whose products are longer, while
      // this warp still publishes: 3 % of the time; with heads of 128 that costs 2 %.)
      if (!STATE_ONLY && kHeads == 2 && c + 1 < n) signal(B_RDY_S, false);
#pragma unroll
      for (int i = 0; i < kCols; i += 2) {
        const float2 r = __ffma2_rn(make_float2(dec, dec), make_float2(s[i], s[i + 1]), make_float2(v[i], v[i + 1]));
        s[i] = r.x;
        s[i + 1] = r.y;
      }
      if (!STATE_ONLY && c + 1 < n) {
        if (met) wait_last(c);  // the product that reads the last published state is done
        publish_state();
        if (kHeads == 1) signal(B_RDY_S, false);
      }
    };

    // (buffer and stage of chunk c + 1, and their parity)
    int st = 0, prev = 0;
    uint32_t st_par = 0;
    for (int c = -1; c < n; ++c) {
      if (__any_sync(0xffffffffu, failed)) {
        failed = true;
        break;
      }
      if (c + 1 < n) {
        if (has_w)
          make_w(c + 1, st, st_par);
        else if (has_m)
          make_m(c + 1, st, st_par);
        else
          wait(B_X + st, st_par);  // (the tables, for the outputs)
      }
      if (c >= 0) {
        update(c, prev);
        if (!STATE_ONLY) outputs(c, prev);
        signal(B_DONE + prev, !STATE_ONLY);
      }
      prev = st;
      if (++st == kStages) {
        st = 0;
        st_par ^= 1u;
      }
    }

    if (!failed) {
      if (STATE_ONLY) {
        const int64_t u = slot * p.tiles + tile;
        float4* F = reinterpret_cast<float4*>(p.ws) + u * (kRows * NS / 4) + tid;
#pragma unroll
        for (int i = 0; i < kCols / 4; ++i)
          F[i * kComputeThreads] = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
        if (cq == 0 && (row & 63) == 0) p.ws_dec[2 * u + (row >> 6)] = dprod;
      }
    }
    if (!STATE_ONLY && last_piece) {
      // (this warp has met the last products that read W and M)
#pragma unroll
      for (int i = 0; i < kCols / 4; ++i) {
        const int col = kCols * cq + 4 * i;
        sts128(state_smem + (col >> 5) * 16384 + (((col >> 2 & 7) ^ (row & 7)) << 4), __float_as_uint(s[4 * i]),
               __float_as_uint(s[4 * i + 1]), __float_as_uint(s[4 * i + 2]), __float_as_uint(s[4 * i + 3]));
      }
      fence_async_smem();
      if (!named_sync_or(kComputeBar, kComputeThreads, failed) && tid == 0) {
#pragma unroll
        for (int cb = 0; cb < NS / 32; ++cb) {
          tma_store_2d(&tm_n, smem + L::OFF_W + cb * 16384, 32 * cb, state_row);
          if (P == 128 || two) tma_store_2d(&tm_n, smem + L::OFF_W + cb * 16384 + 8192, 32 * cb, state_row + 64);
        }
        bulk_commit();
        bulk_wait_read_all();  // (the writes themselves end with the grid)
      }
    }
  } else if (warp == kMmaWarp) {
    // ======================= MMA issue warp ==================================
    constexpr uint32_t idesc_g = idesc_bf16(128, 64, false, false);   // [B; C] B^T
    constexpr uint32_t idesc_ds = idesc_bf16(128, NS, true, true);    // W^T B
    constexpr uint32_t idesc_qs = idesc_bf16(128, 64, false, false);  // S (TMEM) C^T
    constexpr uint32_t idesc_pv = idesc_bf16(128, 64 * kHeads, true, false);   // X^T M^T
    const uint32_t leader = elect_one();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);  // (uniform)
    const uint32_t sb16 = sb >> 4;
    constexpr uint32_t kBcSize16 = L::kBc / 16, kBc16 = L::OFF_BC / 16;
    auto wait = [&](int b, uint32_t parity) -> bool {
      // (inline and without naps: every product waits for this warp; 4 % of the kernel's time)
      const bool done = mbar_wait(&bars[b], parity, kTimeoutNs);
      tc_fence_after();
      return __all_sync(0xffffffffu, done);
    };
    // (bst: the stage of the chunk's B and C, xst: of its x)
    auto mma_g = [&](int bst, uint32_t par) -> bool {
      if (!wait(B_BC + bst, par)) return false;
      const uint32_t bc = sb16 + kBc16 + bst * kBcSize16;
#pragma unroll
      for (int ks = 0; ks < NS / 16; ++ks) {
        const uint64_t d = sdesc_sw128_f(bc + ((ks >> 2) * 16384 + (ks & 3) * 32) / 16, 16, 1024);
        mma_ss_by(leader, tm + TM_G, d, d, idesc_g, ks > 0);
      }
      return true;
    };
    auto mma_ds = [&](int c, int bst) {
      const uint32_t d = tm + TM_DS + (STATE_ONLY ? 128 * (c & 1) : 0), bc = sb16 + kBc16 + bst * kBcSize16;
#pragma unroll
      for (int part = 0; part < kTerms; ++part)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma_ss_by(leader, d, sdesc_sw128_f(sb16 + (L::OFF_W + part * 16384 + ks * 2048) / 16, 8192, 1024),
                    sdesc_sw128_f(bc + ks * 128, 16384, 1024), idesc_ds, part > 0 || ks > 0);
      commit_by(leader, &bars[B_DS + (STATE_ONLY ? c & 1 : 0)]);
    };
    auto mma_pv = [&](int xst) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int term = 0; term < kMTerms; ++term)
          mma_ss_by(leader, tm + TM_PV, sdesc_sw128_f(sb16 + (L::OFF_X + ks * 2048) / 16 + xst * (L::kX / 16), 8192, 1024),
                    sdesc_sw128_f(sb16 + (L::OFF_M + term * L::kM + ks * 32) / 16, 16, 1024), idesc_pv, ks > 0 || term > 0);
      commit_by(leader, &bars[B_PV]);
    };
    auto mma_qs = [&](int bst) {
      const uint32_t bc = sb16 + kBc16 + bst * kBcSize16;
#pragma unroll
      for (int ks = 0; ks < NS / 16; ++ks)
#pragma unroll
        for (int term = 0; term < 2; ++term)
          mma_ts_by(leader, tm + TM_QS, tm + TM_SB + 64 * term + 8 * ks,
                    sdesc_sw128_f(bc + ((ks >> 2) * 16384 + 8192 + (ks & 3) * 32) / 16, 16, 1024), idesc_qs, ks > 0 || term > 0);
      commit_by(leader, &bars[B_QS]);
    };
    bool ok = STATE_ONLY || mma_g(0, 0);
    if (!STATE_ONLY) commit_by(leader, &bars[B_G]);  // (later ones are covered by the commits behind them)
    // stages of chunk c + 1 (of B and C, of x) and of chunk c + 2 (of B and C, with its parity)
    int b1 = 0, x1 = 0, b2 = 1;
    uint32_t par1 = 0, par2 = 0;
    for (int c = -1; ok && c + 1 < n; ++c) {
      const uint32_t next = static_cast<uint32_t>((c + 1) & 1);
      if (STATE_ONLY) {
        // (the buffer of W^T B was read in the update of chunk c - 1)
        if (c >= 1 && !(ok = wait(B_DONE + (c - 1) % kStages, static_cast<uint32_t>(((c - 1) / kStages) & 1)))) break;
        if (!(ok = wait(B_BC + b1, par1))) break;
        if (!(ok = wait(B_RDY_W, next))) break;
        mma_ds(c + 1, b1);
        commit_by(leader, &bars[B_EMPTY + b1]);
      } else {
        if (!(ok = wait(B_RDY_M, next))) break;
        // (G right behind M: the warps that form M wait for it.  After C S it cost 3 %.)
        if (c + 2 < n && !(ok = mma_g(b2, par2))) break;
        if (!(ok = wait(B_RDY_W, next))) break;
        if (!(ok = wait(B_RDY_S, next))) break;  // the update of chunk c has read W^T B
        mma_ds(c + 1, b1);
        // the state that C reads is published and the outputs of chunk c have read their accumulators
        if (c >= 0 && !(ok = wait(B_RDY_D, static_cast<uint32_t>(c & 1)))) break;
        mma_pv(x1);
        mma_qs(b1);
        commit_by(leader, &bars[B_EMPTY + b1]);
      }
      b1 = b2;
      par1 = par2;
      if (++b2 == kBcStages) {
        b2 = 0;
        par2 ^= 1u;
      }
      if (++x1 == kStages) x1 = 0;
    }
    commit_by(leader, &bars[B_END]);
    failed = !wait(B_END, 0) || !ok;
  } else if (warp >= kGateWarp) {
    // ======================= gate tables: warp 18 head 0, warp 19 head 1 =========
    if (gh < kHeads) {
      int buf = 0;
      uint32_t par = 0;
      for (int c = 0; c < n; ++c) {
        const int Lc = live ? static_cast<int>(min(static_cast<int64_t>(kChunk), Ltot - static_cast<int64_t>(c) * kChunk)) : 0;
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
        if (c + 1 < n) load_gates(c + 1);
        const unsigned bad0 = __ballot_sync(0xffffffffu, !ok[0]), bad1 = __ballot_sync(0xffffffffu, !ok[1]);
        const int fb = min(bad0 ? 2 * (__ffs(bad0) - 1) : 64, bad1 ? 2 * (__ffs(bad1) - 1) + 1 : 64);
        // (formed before the tables' places are free)
        float high[2], low[2], u[2], v[2], w[2], eg[2], total;
        unsigned far = 0;
        if constexpr (STATE_ONLY) {  // only W and the chunk's decay: gamma_63 - gamma_t, as sums of their own terms
          float suf = lg[0] + lg[1];
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const float z = __shfl_down_sync(0xffffffffu, suf, d);
            if (lane + d < 32) suf += z;
          }
          const float after = __shfl_down_sync(0xffffffffu, suf, 1);
          const float tail = lane == 31 ? 0.f : after;
          w[0] = dt[0] * ex2_ftz(tail + lg[1]);
          w[1] = dt[1] * ex2_ftz(tail);
          total = suf;
        } else {
          // gamma in 64 bits, and its differences: fp32 sums that a strong decay has made large (the
          // end of a head's memory) would lose the weak ones behind it.  (The fp64 additions are not waited for
          // here; in the first launch, with a chunk in 1 us, they were: +10 % of a call that is cut.)
          double incl = static_cast<double>(lg[0]) + lg[1];
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += y;
          }
          const double gt[2] = {incl - lg[1], incl};
          const double first = __shfl_sync(0xffffffffu, gt[0], lane & 24);
          const double top = __shfl_sync(0xffffffffu, gt[1], lane | 7);
          const double g63 = __shfl_sync(0xffffffffu, gt[1], 31);
          far = __ballot_sync(0xffffffffu, first - top > 64.0);
          auto decay = [](double from, double to) { return ex2_ftz(static_cast<float>(to - from)); };
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            high[e] = static_cast<float>(gt[e]);
            low[e] = static_cast<float>(gt[e] - high[e]);
            u[e] = dt[e] * decay(gt[e], top);
            v[e] = dt[e] * decay(gt[e], first);
            w[e] = dt[e] * decay(gt[e], g63);
            eg[e] = 2 * lane + e >= fb ? __int_as_float(0x7fc00000) : ex2_ftz(high[e]);
          }
          total = static_cast<float>(g63);
        }
        if (c >= kStages && !__all_sync(0xffffffffu, mbar_test(&bars[B_DONE + buf], par ^ 1u)))
          failed = !__all_sync(0xffffffffu, wait_long(&bars[B_DONE + buf], par ^ 1u));
        if (failed) break;
        float* tb = gates + (buf * 2 + gh) * kGateFloats;
        auto put = [&](int table, const float (&x)[2]) {
          *reinterpret_cast<float2*>(tb + table + 2 * lane) = make_float2(x[0], x[1]);
        };
        put(G_W, w);
        if constexpr (!STATE_ONLY) {
          put(G_GAM, high);
          put(G_LOW, low);
          put(G_DT, dt);
          put(G_U, u);
          put(G_V, v);
          put(G_EG, eg);
        }
        if (lane == 0) {
          // (rounded to nearest where it is close to 1: the state is multiplied by it once a chunk, and what the
          // approximation errs to one side would add up)
          decs[buf * 2 + gh] = fb < 64        ? __int_as_float(0x7fc00000)
                               : total > -0.7f ? 1.0f + expm1f(total * kLn2)
                                               : ex2_ftz(total);
          if (!STATE_ONLY) steep[buf * 2 + gh] = (far & 1u) | (far >> 7 & 2u) | (far >> 14 & 4u) | (far >> 21 & 8u);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[B_X + buf]);
        if (++buf == kStages) {
          buf = 0;
          par ^= 1u;
        }
      }
    }
  } else if (lane == 0) {
    // ======================= TMA load and store thread =========================
    bool ok = true;
    for (int c = 0; ok && c < n; ++c) {
      const int st = c % kStages, bst = c % kBcStages;
      const uint32_t par = static_cast<uint32_t>((c / kStages) & 1);
      if (c + kBcStages < n) {
        if (!(ok = mbar_wait(&bars[B_EMPTY + bst], static_cast<uint32_t>((c / kBcStages) & 1), kTimeoutNs))) break;
        load_bc(c + kBcStages);
        if (STATE_ONLY && c + kStages < n) load_x(c + kStages);
      }
      if (STATE_ONLY) continue;
      if (!(ok = mbar_wait(&bars[B_DONE + st], par, kTimeoutNs))) break;
      if (Ltot - static_cast<int64_t>(c) * kChunk >= kChunk) {  // the outputs, where x was
        const int tok = static_cast<int>(bos + static_cast<int64_t>(c) * kChunk);
        const uint8_t* ys = smem + L::OFF_X + st * L::kX;
        tma_store_3d(&tm_y, ys, 0, h0, tok);
        if (P == 128)
          tma_store_3d(&tm_y, ys + 8192, 64, h0, tok);
        else if (two)
          tma_store_3d(&tm_y, ys + 8192, 0, h0 + 1, tok);
        bulk_commit();
      }
      if (c + kStages < n) {
        bulk_wait_read_all();
        load_x(c + kStages);
      }
    }
    // no load may be in flight, and no store may still read, when the CTA ends
    bulk_wait_read_all();
    for (int c = max(0, bc_issued - kBcStages); c < bc_issued; ++c)
      if (!mbar_wait(&bars[B_BC + c % kBcStages], static_cast<uint32_t>((c / kBcStages) & 1), kTimeoutNs)) ok = false;
    for (int c = max(0, x_issued - kStages); c < x_issued; ++c)
      if (!mbar_wait(&bars[B_X + c % kStages], static_cast<uint32_t>((c / kStages) & 1), kTimeoutNs)) ok = false;
    failed = !ok;
  }
  if (failed) atomicOr(&g_ssm_status, kStatusSsmTimeout);
  __syncwarp();
  if (ends_last) dependency_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---- host side ---------------------------------------------------------------
// [T, heads, inner] bf16, box = 64 tokens x 1 head x 64 values, or (heads = 0) [T, inner] fp32,
// box = 64 rows x 32 values; 128-byte swizzle.
cudaError_t encode_map(CUtensorMap* m, const void* base, int64_t inner, int64_t heads, int64_t T) {
  auto fn = tmap_encoder();
  if (!fn) return cudaErrorNotSupported;
  const bool tokens = heads != 0;
  const cuuint64_t n = static_cast<cuuint64_t>(inner), h = static_cast<cuuint64_t>(heads), t = static_cast<cuuint64_t>(T);
  const cuuint64_t dims[3] = {n, tokens ? h : t, t}, strides[2] = {n * (tokens ? 2 : 4), h * n * 2};
  const cuuint32_t box[3] = {tokens ? 64u : 32u, tokens ? 1u : 64u, 64}, es[3] = {1, 1, 1};
  const CUresult r = fn(m, tokens ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, tokens ? 3 : 2,
                        const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t make_map(CUtensorMap* m, const void* base, int64_t inner, int64_t heads, int64_t T) {
  return cached_tmap(m, {base, {inner, heads, T}},
                     [=](CUtensorMap* map) { return encode_map(map, base, inner, heads, T); });
}

int64_t head_tiles(int64_t H, int64_t G, int64_t P) { return G * ((H / G * P + kRows - 1) / kRows); }

struct Cut {
  int64_t seg = 0;    // tokens of a piece, 0: no cut
  int64_t slots = 0;  // at most so many pieces
};

// Times in units of one chunk of the second launch on one SM (~2.5 us): a chunk of the first,
// the start and end of a CTA, the state of one earlier piece, a launch.
constexpr double kStateChunk = 0.4, kCta = 3.0, kJoin = 0.3, kLaunch = 1.5;

// Only the mean length is known here (the lengths lie on the device): the piece length is the
// one that is best for sequences of that length.  Calls that fill the SMs with whole sequences
// are cut too, but only sequences of twice the work of an SM, which would run on alone for most
// of the call; where there are none, the first launch and the search cost ~4 us.  That is done where a
// sequence of that length is either likely (twice the mean) or a small part of the call (a quarter), so that
// cutting it gains much.  Measured, whole | cut, 64 heads of 64 unless said: 4 sequences, 65536 tokens,
// even 699 | 701 us, ragged 1272 | 1131, half the tokens in one 1634 | 1125; 128 sequences, 16384
// tokens, 32 heads, even 155 | 156, half in one 380 | 228.  Not done: 16 sequences, 7648 tokens, even
// 111 | 115, ragged 120 | 123, half in one 190 | 147.
Cut choose_cut(int64_t T, int64_t N, int64_t tiles, int sms) {
  const int64_t chunks = std::max<int64_t>(1, (T + N * kChunk - 1) / (N * kChunk));  // of a mean sequence
  auto waves = [&](int64_t ctas) { return static_cast<double>((ctas + sms - 1) / sms); };
  Cut best{0, N};
  double best_time = waves(N * tiles) * (chunks + kCta);
  for (int64_t p = 2; p <= 64 && p <= chunks; ++p) {
    const int64_t seg = (chunks + p - 1) / p;
    if (seg < 2) break;
    const int64_t pieces = (chunks + seg - 1) / seg;
    const double time = waves(N * (pieces - 1) * tiles) * (seg * kStateChunk + kCta) + kLaunch +
                        waves(N * pieces * tiles) * (seg + kCta + kJoin * (pieces - 1) / 2);
    if (time < 0.9 * best_time) {
      best_time = time;
      best.seg = seg;
    }
  }
  const int64_t all = T / kChunk, share = (all * tiles + sms - 1) / sms;  // chunks of an SM, were they spread evenly
  const int64_t longest = std::max(2 * share, chunks + 1);
  if (best.seg == 0 && all >= 64 && 2 * longest <= all && (longest <= 2 * chunks || 4 * longest <= all)) best.seg = longest;
  if (best.seg) {
    best.seg *= kChunk;
    best.slots = N + T / best.seg;  // the pieces of N sequences of T tokens are at most this many
  }
  return best;
}

template <int P, int NS, bool STATE_ONLY>
cudaError_t launch_one(const CUtensorMap* m, const Params& p, int64_t slots, bool overlap, cudaStream_t s) {
  auto kernel = gdn_ssm_chunked_kernel<P, NS, STATE_ONLY>;
  constexpr int bytes = Lay<P, NS>::kBytes;
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess) return e;
  const int64_t ctas = slots * p.tiles;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, m[0], m[1], m[2], m[3], m[4], m[5], p);
}

template <int P, int NS>
cudaError_t launch(const SsmArgs& a, const Cut& cut, void* ws, cudaStream_t s) {
  CUtensorMap m[6];
  memset(m, 0, sizeof(m));
  cudaError_t e;
  if ((e = make_map(&m[0], a.x, P, a.H, a.T)) != cudaSuccess) return e;
  if ((e = make_map(&m[1], a.B, NS, a.G, a.T)) != cudaSuccess) return e;
  if ((e = make_map(&m[2], a.C, NS, a.G, a.T)) != cudaSuccess) return e;
  if ((e = make_map(&m[3], a.out, P, a.H, a.T)) != cudaSuccess) return e;
  if (a.state && (e = make_map(&m[4], a.state, NS, 0, a.N * a.H * P)) != cudaSuccess) return e;
  if ((e = make_map(&m[5], a.new_state, NS, 0, a.N * a.H * P)) != cudaSuccess) return e;
  Params p{a.state, a.A_log, a.dt_bias, a.D, static_cast<const __nv_bfloat16*>(a.a), a.cu_seqlens,
           static_cast<__nv_bfloat16*>(a.out), a.new_state, static_cast<float*>(ws), nullptr, a.T, a.N, cut.seg, cut.slots - a.N,
           static_cast<int>(a.H), static_cast<int>(a.G), static_cast<int>(head_tiles(a.H, a.G, P))};
  if (cut.seg) {
    p.ws_dec = p.ws + p.inner * p.tiles * kRows * NS;
    if (p.inner > 0) {
      if ((e = launch_one<P, NS, true>(m, p, p.inner, false, s)) != cudaSuccess) return e;
      return launch_one<P, NS, false>(m, p, cut.slots, true, s);
    }
  }
  return launch_one<P, NS, false>(m, p, cut.slots, false, s);
}

}  // namespace

size_t ssm_chunked_workspace(int64_t T, int64_t N, int64_t H, int64_t G, int64_t P, int64_t Ns, int sms) {
  const int64_t tiles = head_tiles(H, G, P);
  const Cut cut = choose_cut(T, N, tiles, sms);
  return cut.seg ? static_cast<size_t>(cut.slots - N) * tiles * (kRows * Ns + 2) * sizeof(float) : 0;
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
