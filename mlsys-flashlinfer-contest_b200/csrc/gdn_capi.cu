// C ABI of the gdn_b200 library: validation, dispatch and error reporting.
// Declarations and the contract of each entry point: include/gdn_b200.h.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include "../../include/gdn_b200.h"
#include "gdn_internal.h"

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int ok() {
  g_err[0] = '\0';
  return GDN_OK;
}

int cuda_status(cudaError_t e, const char* what) {
  if (e != cudaSuccess) return fail(GDN_ERR_CUDA, "%s failed: %s", what, cudaGetErrorString(e));
  return ok();
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

// [p, p+bytes) and [q, q+bytes) overlap without being identical
bool partial_overlap(const void* p, const void* q, size_t bytes) {
  if (p == nullptr || q == nullptr || p == q) return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return a < b + bytes && b < a + bytes;
}

int check_heads(int64_t Hq, int64_t Hk, int64_t Hv, int64_t D) {
  if (D != gdn::kHead) return fail(GDN_ERR_VALUE, "head_size must be 128 (got %lld)", (long long)D);
  if (Hq <= 0 || Hk <= 0) return fail(GDN_ERR_VALUE, "head counts must be positive");
  if (Hk != Hq)
    return fail(GDN_ERR_VALUE, "num_k_heads (%lld) must equal num_q_heads (%lld)", (long long)Hk,
                (long long)Hq);
  if (Hv < Hq || Hv % Hq != 0)
    return fail(GDN_ERR_VALUE, "num_v_heads (%lld) must be a multiple of num_q_heads (%lld)",
                (long long)Hv, (long long)Hq);
  return GDN_OK;
}

int64_t upper_bound_chunks(int64_t T, int64_t N) {
  if (T <= 0 || N <= 0) return 0;
  if (T < N) return T;
  return N + (T - N) / gdn::kChunk;
}

}  // namespace

extern "C" {

int gdn_abi_version(void) { return GDN_ABI_VERSION; }

const char* gdn_last_error(void) { return g_err; }

int64_t gdn_chunk_upper_bound(int64_t T, int64_t N) { return upper_bound_chunks(T, N); }

int gdn_decode(const void* q, const void* k, const void* v, const float* state, const float* A_log,
               const void* a, const float* dt_bias, const void* b, float scale, void* output,
               float* new_state, int64_t B, int64_t Hq, int64_t Hk, int64_t Hv, int64_t D,
               void* stream) {
  if (int e = check_heads(Hq, Hk, Hv, D)) return e;
  if (B < 0) return fail(GDN_ERR_VALUE, "batch_size must be non-negative");
  if (B == 0) return ok();
  if (!q || !k || !v || !A_log || !a || !dt_bias || !b || !output || !new_state)
    return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(q, 8) || !aligned(k, 8))
    return fail(GDN_ERR_VALUE, "q and k must be 8-byte aligned");
  if (!aligned(new_state, 16) || (state && !aligned(state, 16)))
    return fail(GDN_ERR_VALUE, "state and new_state must be 16-byte aligned");
  const size_t state_bytes = static_cast<size_t>(B) * Hv * gdn::kHead * gdn::kHead * 4;
  if (partial_overlap(state, new_state, state_bytes))
    return fail(GDN_ERR_VALUE, "new_state overlaps state without being the same buffer");
  gdn::DecodeArgs p{q, k, v, state, A_log, a, dt_bias, b, scale == 0.0f ? 0.08838834764831845f : scale,
                    output, new_state, B, Hq, Hv};
  return cuda_status(gdn::launch_decode(p, 0, static_cast<cudaStream_t>(stream)), "gdn_decode launch");
}

int gdn_decode_pool(const void* q, const void* k, const void* v, const float* A_log, const void* a,
                    const float* dt_bias, const void* b, float scale, void* pool, int state_dtype,
                    int64_t pool_size, const int32_t* in_slots, const int32_t* out_slots,
                    void* intermediate, int flags, void* output, int64_t B, int64_t T, int64_t Hq,
                    int64_t Hk, int64_t Hv, int64_t D, void* stream) {
  if (int e = check_heads(Hq, Hk, Hv, D)) return e;
  if (B < 0) return fail(GDN_ERR_VALUE, "batch_size must be non-negative");
  if (T < 1) return fail(GDN_ERR_VALUE, "seq_len must be at least 1");
  if (pool_size < 0) return fail(GDN_ERR_VALUE, "pool_size must be non-negative");
  if (pool_size > INT32_MAX) return fail(GDN_ERR_VALUE, "pool_size must fit int32 slot indices");
  if (state_dtype != GDN_STATE_F32 && state_dtype != GDN_STATE_BF16)
    return fail(GDN_ERR_TYPE, "state_dtype must be GDN_STATE_F32 or GDN_STATE_BF16");
  if (flags & ~(GDN_POOL_QK_L2NORM | GDN_POOL_NO_STATE_UPDATE))
    return fail(GDN_ERR_VALUE, "unknown flags");
  if (B == 0) return ok();
  if (!q || !k || !v || !A_log || !a || !dt_bias || !b || !output || !in_slots)
    return fail(GDN_ERR_VALUE, "null pointer argument");
  if (pool_size > 0 && !pool) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(pool, 16) ||
      !aligned(intermediate, 16))
    return fail(GDN_ERR_VALUE, "q, k, v, state_pool and intermediate must be 16-byte aligned");
  if (!aligned(in_slots, 4) || !aligned(out_slots, 4))
    return fail(GDN_ERR_VALUE, "slot arrays must be 4-byte aligned");
  gdn::DecodePoolArgs p{q, k, v, A_log, a, dt_bias, b, scale == 0.0f ? 0.08838834764831845f : scale,
                        pool, in_slots, out_slots, intermediate, output, B, T, Hq, Hv, pool_size,
                        state_dtype == GDN_STATE_BF16, (flags & GDN_POOL_QK_L2NORM) != 0,
                        (flags & GDN_POOL_NO_STATE_UPDATE) != 0};
  return cuda_status(gdn::launch_decode_pool(p, static_cast<cudaStream_t>(stream)),
                     "gdn_decode_pool launch");
}

static int check_prefill(const void* q, const void* k, const void* v, const float* state,
                         const float* A_log, const void* a, const float* dt_bias, const void* b,
                         const int64_t* cu, void* out, float* new_state, int64_t T, int64_t N,
                         int64_t Hq, int64_t Hk, int64_t Hv, int64_t D) {
  if (int e = check_heads(Hq, Hk, Hv, D)) return e;
  if (N <= 0) return fail(GDN_ERR_VALUE, "must have at least one sequence");
  if (T < 0) return fail(GDN_ERR_VALUE, "total_seq_len must be non-negative");
  if (!cu || !A_log || !dt_bias || !new_state) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (T > 0 && (!q || !k || !v || !a || !b || !out)) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16))
    return fail(GDN_ERR_VALUE, "q, k and v must be 16-byte aligned");
  if (!aligned(new_state, 16) || (state && !aligned(state, 16)))
    return fail(GDN_ERR_VALUE, "state and new_state must be 16-byte aligned");
  if (!aligned(cu, 8)) return fail(GDN_ERR_VALUE, "cu_seqlens must be 8-byte aligned");
  const size_t state_bytes = static_cast<size_t>(N) * Hv * gdn::kHead * gdn::kHead * 4;
  if (partial_overlap(state, new_state, state_bytes))
    return fail(GDN_ERR_VALUE, "new_state overlaps state without being the same buffer");
  return GDN_OK;
}

int gdn_prefill_recurrent(const void* q, const void* k, const void* v, const float* state,
                          const float* A_log, const void* a, const float* dt_bias, const void* b,
                          const int64_t* cu_seqlens, float scale, void* output, float* new_state,
                          int64_t T, int64_t N, int64_t Hq, int64_t Hk, int64_t Hv, int64_t D,
                          void* stream) {
  if (int e = check_prefill(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, output, new_state, T,
                            N, Hq, Hk, Hv, D))
    return e;
  gdn::PrefillArgs p{q, k, v, state, A_log, a, dt_bias, b, cu_seqlens,
                     scale == 0.0f ? 0.08838834764831845f : scale, output, new_state, T, N, Hq, Hv};
  return cuda_status(gdn::launch_prefill_recurrent(p, static_cast<cudaStream_t>(stream)),
                     "gdn_prefill_recurrent launch");
}

// Chooses the token-recurrent kernel for tiny inputs and the fused chunked
// kernel otherwise.  The reference dispatches on the same two sizes
// (gdn_prefill/solution/python/gdn_prefill_mix.py:29: N <= 2 and T <= 30 N);
// the bounds here come from timing both kernels on a B200 over N = 1..32
// sequences of 8..512 tokens (Hv = 8 and 32): the recurrent kernel walks one
// token at a time (~0.3 us each) while the chunked kernel's floor is one chunk
// (~14.5 us per call, launch included).  Recurrent wins for sequences of up to
// ~32 tokens when there are at most 16 (sequence, head) pairs, up to 16 tokens
// at up to 64 pairs, and up to 8 tokens at any count.  The last bound also caps
// T, because only the mean length is known on the host: one long sequence among
// many short ones walks all its tokens.
static bool use_recurrent(int64_t T, int64_t N, int64_t Hv) {
  return (T <= 32 * N && N * Hv <= 16) || (T <= 16 * N && N * Hv <= 64) ||
         (T <= 8 * N && T <= 256);
}

// Upper bound on the piece count of the sequence-parallel prefill (1: one chain
// per (sequence, head)).  The job builder picks each sequence's count under it
// from the lengths on the device (the shortest longest chain whose passes fit the
// SMs: pass 1 within one to three waves of the SMs its piece-0 jobs leave free,
// pass 2 within one wave), so the host only rules out calls that cannot gain:
// more (sequence, head) pairs than half the SMs (then not even equal sequences
// could all be cut in 3 with pass 2 in one wave), or fewer chunks in all than
// the shortest sequence the builder would cut (prefill_min_cut_chunks); the
// bound is the largest G <= kMaxAutoSegments with N Hv (G - 1) <= 2 SMs and
// T >= 4 G chunks.
static int sm_count() { return gdn::device_sm_count(); }
constexpr int kMaxAutoSegments = 16;

static int choose_segments(int64_t T, int64_t N, int64_t Hv) {
  if (N <= 0 || Hv <= 0 || 2 * N * Hv > sm_count()) return 1;
  const int64_t chunks = T / gdn::kChunk;
  // no sequence can be long enough for the builder to accept a cut: the
  // segmented form would only add its launches
  if ((T + gdn::kChunk - 1) / gdn::kChunk < gdn::prefill_min_cut_chunks()) return 1;
  int best = 1;
  for (int G = 3; G <= kMaxAutoSegments; ++G)
    if (N * Hv * (G - 1) <= 2 * sm_count() && chunks >= 4 * G) best = G;
  return best;
}

int gdn_prefill_segments(int64_t T, int64_t N, int64_t Hv) {
  return use_recurrent(T, N, Hv) ? 1 : choose_segments(T, N, Hv);
}

// segments 0: the automatic form (sized for the largest bound)
size_t gdn_prefill_segmented_workspace_bytes(int64_t N, int64_t Hv, int segments) {
  if (segments == 0) return gdn::prefill_segments_bytes(N, Hv, kMaxAutoSegments, true, sm_count());
  return gdn::prefill_segments_bytes(N, Hv, segments, false, sm_count());
}

size_t gdn_prefill_workspace_bytes(int64_t T, int64_t N, int64_t Hq, int64_t Hv) {
  (void)Hq;
  const int G = gdn_prefill_segments(T, N, Hv);
  return G > 1 ? gdn::prefill_segments_bytes(N, Hv, G, true, sm_count()) : 0;
}

int gdn_prefill_chunked(const void* q, const void* k, const void* v, const float* state,
                        const float* A_log, const void* a, const float* dt_bias, const void* b,
                        const int64_t* cu_seqlens, float scale, void* output, float* new_state,
                        int64_t T, int64_t N, int64_t Hq, int64_t Hk, int64_t Hv, int64_t D,
                        void* stream) {
  if (int e = check_prefill(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, output, new_state, T,
                            N, Hq, Hk, Hv, D))
    return e;
  if (T > 0x7fffffffLL - 64) return fail(GDN_ERR_VALUE, "total_seq_len too large");
  gdn::PrefillArgs p{q, k, v, state, A_log, a, dt_bias, b, cu_seqlens,
                     scale == 0.0f ? 0.08838834764831845f : scale, output, new_state, T, N, Hq, Hv};
  return cuda_status(gdn::launch_prefill_chunked(p, static_cast<cudaStream_t>(stream)),
                     "gdn_prefill_chunked launch");
}

int gdn_prefill(const void* q, const void* k, const void* v, const float* state, const float* A_log,
                const void* a, const float* dt_bias, const void* b, const int64_t* cu_seqlens,
                float scale, void* output, float* new_state, int64_t T, int64_t N, int64_t Hq,
                int64_t Hk, int64_t Hv, int64_t D, void* workspace, size_t workspace_bytes,
                void* stream) {
  if (use_recurrent(T, N, Hv))
    return gdn_prefill_recurrent(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, scale, output,
                                 new_state, T, N, Hq, Hk, Hv, D, stream);
  const int G = choose_segments(T, N, Hv);
  if (G > 1 && workspace && workspace_bytes >= gdn::prefill_segments_bytes(N, Hv, G, true, sm_count()))
    return gdn_prefill_segmented(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, scale, output,
                                 new_state, T, N, Hq, Hk, Hv, D, 0, 0, workspace, workspace_bytes,
                                 stream);
  return gdn_prefill_chunked(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, scale, output,
                             new_state, T, N, Hq, Hk, Hv, D, stream);
}

// Checks shared by the segmented entries; segments 0 = automatic (an upper bound
// for the device's per-sequence choice).
static int segmented_setup(int64_t T, int64_t N, int64_t Hv, int* segments, bool* adaptive,
                           void* workspace, size_t workspace_bytes) {
  if (*segments < 0 || *segments > 64) return fail(GDN_ERR_VALUE, "segments must be in [0, 64]");
  *adaptive = *segments == 0;
  if (*adaptive) *segments = choose_segments(T, N, Hv);
  const size_t need = gdn::prefill_segments_bytes(N, Hv, *segments, *adaptive, sm_count());
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(GDN_ERR_VALUE, "workspace needs %zu bytes", need);
  if (!aligned(workspace, 256)) return fail(GDN_ERR_VALUE, "workspace must be 256-byte aligned");
  return GDN_OK;
}

int gdn_prefill_segmented(const void* q, const void* k, const void* v, const float* state,
                          const float* A_log, const void* a, const float* dt_bias, const void* b,
                          const int64_t* cu_seqlens, float scale, void* output, float* new_state,
                          int64_t T, int64_t N, int64_t Hq, int64_t Hk, int64_t Hv, int64_t D,
                          int flags, int segments, void* workspace, size_t workspace_bytes,
                          void* stream) {
  if (flags & ~GDN_PREFILL_QK_L2NORM) return fail(GDN_ERR_VALUE, "unknown flags");
  if (int e = check_prefill(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, output, new_state, T,
                            N, Hq, Hk, Hv, D))
    return e;
  if (T > 0x7fffffffLL - 64) return fail(GDN_ERR_VALUE, "total_seq_len too large");
  bool adaptive = false;
  if (int e = segmented_setup(T, N, Hv, &segments, &adaptive, workspace, workspace_bytes)) return e;
  gdn::PrefillArgs p{q, k, v, state, A_log, a, dt_bias, b, cu_seqlens,
                     scale == 0.0f ? 0.08838834764831845f : scale, output, new_state, T, N, Hq, Hv,
                     (flags & GDN_PREFILL_QK_L2NORM) != 0};
  return cuda_status(gdn::launch_prefill_segmented(p, segments, adaptive, sm_count(), workspace,
                                                   workspace_bytes, static_cast<cudaStream_t>(stream)),
                     "gdn_prefill_segmented launch");
}

int gdn_prefill_ex(const void* q, const void* k, const void* v, const float* state,
                   const float* A_log, const void* a, const float* dt_bias, const void* b,
                   const int64_t* cu_seqlens, float scale, void* output, float* new_state, int64_t T,
                   int64_t N, int64_t Hq, int64_t Hk, int64_t Hv, int64_t D, int flags, int path,
                   void* stream) {
  if (flags & ~GDN_PREFILL_QK_L2NORM) return fail(GDN_ERR_VALUE, "unknown flags");
  if (path < GDN_PREFILL_PATH_AUTO || path > GDN_PREFILL_PATH_CHUNKED)
    return fail(GDN_ERR_VALUE, "unknown path");
  if (int e = check_prefill(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, output, new_state, T,
                            N, Hq, Hk, Hv, D))
    return e;
  if (T > 0x7fffffffLL - 64) return fail(GDN_ERR_VALUE, "total_seq_len too large");
  gdn::PrefillArgs p{q, k, v, state, A_log, a, dt_bias, b, cu_seqlens,
                     scale == 0.0f ? 0.08838834764831845f : scale, output, new_state, T, N, Hq, Hv,
                     (flags & GDN_PREFILL_QK_L2NORM) != 0};
  const bool recurrent =
      path == GDN_PREFILL_PATH_RECURRENT || (path == GDN_PREFILL_PATH_AUTO && use_recurrent(T, N, Hv));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return recurrent ? cuda_status(gdn::launch_prefill_recurrent(p, st), "gdn_prefill_recurrent launch")
                   : cuda_status(gdn::launch_prefill_chunked(p, st), "gdn_prefill_chunked launch");
}

// No-allocation form of gdn_prefill_segmented: the scratch is the library's own
// device array (gdn::kNoAllocScratchBytes per GPU), whose address on the current
// device is looked up on the first call on that device.
int gdn_prefill_segmented_noalloc(const void* q, const void* k, const void* v, const float* state,
                                  const float* A_log, const void* a, const float* dt_bias,
                                  const void* b, const int64_t* cu_seqlens, float scale,
                                  void* output, float* new_state, int64_t T, int64_t N, int64_t Hq,
                                  int64_t Hk, int64_t Hv, int64_t D, int flags, int segments,
                                  void* stream) {
  static_assert(GDN_NOALLOC_SCRATCH_BYTES == gdn::kNoAllocScratchBytes, "scratch size");
  if (flags & ~GDN_PREFILL_QK_L2NORM) return fail(GDN_ERR_VALUE, "unknown flags");
  if (int e = check_prefill(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, output, new_state, T,
                            N, Hq, Hk, Hv, D))
    return e;
  if (T > 0x7fffffffLL - 64) return fail(GDN_ERR_VALUE, "total_seq_len too large");
  if (segments < 0 || segments > 64) return fail(GDN_ERR_VALUE, "segments must be in [0, 64]");
  const bool adaptive = segments == 0;
  if (adaptive) segments = choose_segments(T, N, Hv);
  const size_t need = gdn::prefill_segments_bytes(N, Hv, segments, adaptive, sm_count());
  if (need > gdn::kNoAllocScratchBytes)
    return fail(GDN_ERR_VALUE,
                "%lld sequences x %lld heads in %d pieces need %zu bytes of scratch; the "
                "no-allocation entry holds %zu (use gdn_prefill_segmented with a workspace)",
                static_cast<long long>(N), static_cast<long long>(Hv), segments, need,
                gdn::kNoAllocScratchBytes);
  gdn::PrefillArgs p{q, k, v, state, A_log, a, dt_bias, b, cu_seqlens,
                     scale == 0.0f ? 0.08838834764831845f : scale, output, new_state, T, N, Hq, Hv,
                     (flags & GDN_PREFILL_QK_L2NORM) != 0};
  return cuda_status(gdn::launch_prefill_segmented_noalloc(p, segments, adaptive, sm_count(),
                                                           static_cast<cudaStream_t>(stream)),
                     "gdn_prefill_segmented_noalloc launch");
}

int gdn_prefill_chunked_peers(const void* q, const void* k, const void* v, const float* state,
                              const float* A_log, const void* a, const float* dt_bias, const void* b,
                              const int64_t* cu_seqlens, float scale, void* output, float* new_state,
                              int64_t T, int64_t N, int64_t Hq, int64_t Hk, int64_t Hv, int64_t D,
                              int64_t Hv_out, int64_t head_offset, void* const* peer_outputs,
                              int num_peers, int segments, void* workspace, size_t workspace_bytes,
                              void* stream) {
  if (int e = check_prefill(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, output, new_state, T,
                            N, Hq, Hk, Hv, D))
    return e;
  if (T > 0x7fffffffLL - 64) return fail(GDN_ERR_VALUE, "total_seq_len too large");
  if (num_peers < 0 || num_peers > gdn::kMaxPeers)
    return fail(GDN_ERR_VALUE, "num_peers must be in [0, %d]", gdn::kMaxPeers);
  if (num_peers > 0 && !peer_outputs) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (head_offset < 0 || Hv_out < Hv || head_offset + Hv > Hv_out || Hv_out > 0x7fffffffLL)
    return fail(GDN_ERR_VALUE, "heads [head_offset, head_offset + num_v_heads) must lie in the output");
  if (!aligned(output, 16)) return fail(GDN_ERR_VALUE, "output must be 16-byte aligned");
  for (int r = 0; r < num_peers; ++r)
    if (!peer_outputs[r] || !aligned(peer_outputs[r], 16))
      return fail(GDN_ERR_VALUE, "peer output %d is null or not 16-byte aligned", r);
  bool adaptive = false;
  if (int e = segmented_setup(T, N, Hv, &segments, &adaptive, workspace, workspace_bytes)) return e;
  gdn::PrefillArgs p{q, k, v, state, A_log, a, dt_bias, b, cu_seqlens,
                     scale == 0.0f ? 0.08838834764831845f : scale, output, new_state, T, N, Hq, Hv};
  p.out_heads = Hv_out;
  p.out_head_off = head_offset;
  p.n_peers = num_peers;
  p.peer_out = peer_outputs;
  return cuda_status(gdn::launch_prefill_segmented(p, segments, adaptive, sm_count(), workspace,
                                                   workspace_bytes, static_cast<cudaStream_t>(stream)),
                     "gdn_prefill_chunked_peers launch");
}

int gdn_prefill_chunked_debug(const void* q, const void* k, const void* v, const float* state,
                              const float* A_log, const void* a, const float* dt_bias,
                              const void* b, const int64_t* cu_seqlens, float scale, void* output,
                              float* new_state, int64_t T, int64_t N, int64_t Hq, int64_t Hk,
                              int64_t Hv, int64_t D, float* debug, int64_t debug_floats,
                              int64_t dbg_seq, int64_t dbg_head, int64_t dbg_chunk, void* stream) {
  if (int e = check_prefill(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, output, new_state, T,
                            N, Hq, Hk, Hv, D))
    return e;
  if (!debug || debug_floats < gdn::prefill_chunked_debug_floats())
    return fail(GDN_ERR_VALUE, "debug buffer needs %d floats", gdn::prefill_chunked_debug_floats());
  gdn::PrefillArgs p{q, k, v, state, A_log, a, dt_bias, b, cu_seqlens,
                     scale == 0.0f ? 0.08838834764831845f : scale, output, new_state, T, N, Hq, Hv};
  return cuda_status(
      gdn::launch_prefill_chunked_debug(p, debug, static_cast<int>(dbg_seq),
                                        static_cast<int>(dbg_head), static_cast<int>(dbg_chunk),
                                        static_cast<cudaStream_t>(stream)),
      "gdn_prefill_chunked_debug launch");
}

int64_t gdn_prefill_chunked_debug_floats(void) { return gdn::prefill_chunked_debug_floats(); }

int gdn_read_status(uint32_t* status, int clear) {
  if (!status) return fail(GDN_ERR_VALUE, "null pointer argument");
  return cuda_status(gdn::read_status(status, clear != 0), "gdn_read_status");
}

int gdn_wait_probe(uint64_t timeout_ns, uint32_t* result, void* stream) {
  if (timeout_ns > 5000000000ull) return fail(GDN_ERR_VALUE, "timeout_ns must be <= 5 s");
  return cuda_status(gdn::launch_wait_probe(timeout_ns, result, static_cast<cudaStream_t>(stream)),
                     "gdn_wait_probe launch");
}

int gdn_prep_meta(const int64_t* cu_seqlens, int64_t N, int32_t* chunk_offsets,
                  int32_t* chunk_indices, int64_t max_chunks, void* stream) {
  if (N < 0) return fail(GDN_ERR_VALUE, "num_seqs must be non-negative");
  if (!cu_seqlens || !chunk_offsets || (max_chunks > 0 && !chunk_indices))
    return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(chunk_indices, 8)) return fail(GDN_ERR_VALUE, "chunk_indices must be 8-byte aligned");
  return cuda_status(gdn::launch_prep_meta(cu_seqlens, N, chunk_offsets, chunk_indices, max_chunks,
                                           static_cast<cudaStream_t>(stream)),
                     "gdn_prep_meta launch");
}

// Byte ranges [p, p + np) and [q, q + nq) share a byte.
static bool overlap(const void* p, size_t np, const void* q, size_t nq) {
  if (!p || !q || !np || !nq) return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return a < b + nq && b < a + np;
}

struct Range {
  const void* p;
  size_t bytes;
};
// One of the ranges that are written shares a byte with another of them or with one that is read.
static bool any_overlap(const Range* written, int nw, const Range* read, int nr) {
  for (int i = 0; i < nw; ++i) {
    for (int j = i + 1; j < nw; ++j)
      if (overlap(written[i].p, written[i].bytes, written[j].p, written[j].bytes)) return true;
    for (int j = 0; j < nr; ++j)
      if (overlap(written[i].p, written[i].bytes, read[j].p, read[j].bytes)) return true;
  }
  return false;
}

// The outputs of a convolution of `rows` rows, and `extra` that it writes too, against what it reads
// (x spans x_elems elements; the neighbours' rows are read while a row is written).
static bool conv_overlap(const gdn::ConvArgs& a, int64_t rows, int64_t x_elems, Range extra, const void* state) {
  Range w[gdn::kMaxConvOutputs + 1];
  for (int i = 0; i < a.out.count; ++i) w[i] = {a.out.ptr[i], static_cast<size_t>(rows) * a.out.width[i] * 2};
  w[a.out.count] = extra;
  const size_t wide = static_cast<size_t>(a.D) * 2;
  const Range r[4] = {{a.x, rows ? static_cast<size_t>(x_elems) * 2 : 0}, {a.weight, wide * a.W}, {a.bias, wide},
                      {state, extra.bytes}};
  return any_overlap(w, a.out.count + 1, r, 4);
}

static int check_conv(const void* x, int64_t x_batch, int64_t x_row, const void* weight, const void* bias,
                      void* const* outputs, const int64_t* widths, int count, int64_t T, int64_t N,
                      int64_t D, int64_t W, int dtype, int flags, gdn::ConvArgs* a) {
  if (W < 2 || W > 4) return fail(GDN_ERR_VALUE, "width must be 2, 3 or 4 (got %lld)", (long long)W);
  if (D <= 0 || D % 8 != 0)
    return fail(GDN_ERR_VALUE, "dim must be a positive multiple of 8 (got %lld)", (long long)D);
  if (T < 0 || N < 0) return fail(GDN_ERR_VALUE, "lengths and counts must be non-negative");
  if (dtype != GDN_BF16 && dtype != GDN_F16) return fail(GDN_ERR_TYPE, "dtype must be GDN_BF16 or GDN_F16");
  if (flags & ~GDN_CONV_SILU) return fail(GDN_ERR_VALUE, "unknown flags");
  if (count < 1 || count > gdn::kMaxConvOutputs)
    return fail(GDN_ERR_VALUE, "num_outputs must be in [1, %d]", gdn::kMaxConvOutputs);
  if (!weight || !outputs || !widths || (T > 0 && !x)) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (x_row < D || x_row % 8 != 0 || x_batch < 0 || x_batch % 8 != 0)
    return fail(GDN_ERR_VALUE, "x strides must be multiples of 8 and rows at least dim apart");
  if (!aligned(x, 16) || !aligned(weight, 16) || !aligned(bias, 16))
    return fail(GDN_ERR_VALUE, "x, weight and bias must be 16-byte aligned");
  int64_t sum = 0;
  for (int i = 0; i < count; ++i) {
    if (widths[i] <= 0 || widths[i] % 8 != 0)
      return fail(GDN_ERR_VALUE, "output widths must be positive multiples of 8");
    if ((T > 0 && !outputs[i]) || !aligned(outputs[i], 16))
      return fail(GDN_ERR_VALUE, "output %d is null or not 16-byte aligned", i);
    a->out.ptr[i] = outputs[i];
    a->out.width[i] = widths[i];
    sum += widths[i];
  }
  if (sum != D) return fail(GDN_ERR_VALUE, "output widths must sum to dim");
  a->out.count = count;
  a->x = x;
  a->weight = weight;
  a->bias = bias;
  a->x_batch_stride = x_batch;
  a->x_row_stride = x_row;
  a->T = T;
  a->N = N;
  a->D = D;
  a->W = W;
  a->fp16 = dtype == GDN_F16;
  a->silu = (flags & GDN_CONV_SILU) != 0;
  return GDN_OK;
}

int gdn_conv(const void* x, int64_t x_row_stride, const void* weight, const void* bias, const void* state,
             const int64_t* cu_seqlens, void* const* outputs, const int64_t* widths, int num_outputs,
             void* new_state, int64_t T, int64_t N, int64_t D, int64_t W, int dtype, int flags,
             void* stream) {
  gdn::ConvArgs a{};
  if (N <= 0) return fail(GDN_ERR_VALUE, "must have at least one sequence");
  if (int e = check_conv(x, 0, x_row_stride, weight, bias, outputs, widths, num_outputs, T, N, D, W, dtype,
                         flags, &a))
    return e;
  if (!cu_seqlens || !new_state) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(state, 16) || !aligned(new_state, 16) || !aligned(cu_seqlens, 8))
    return fail(GDN_ERR_VALUE, "state and new_state must be 16-byte and cu_seqlens 8-byte aligned");
  const size_t bytes = static_cast<size_t>(N) * (W - 1) * D * 2;
  if (overlap(state, bytes, new_state, bytes)) return fail(GDN_ERR_VALUE, "new_state overlaps state");
  if (conv_overlap(a, T, (T - 1) * x_row_stride + D, {new_state, bytes}, state))
    return fail(GDN_ERR_VALUE, "an output overlaps another tensor");
  a.state = state;
  a.new_state = new_state;
  a.cu_seqlens = cu_seqlens;
  return cuda_status(gdn::launch_conv(a, static_cast<cudaStream_t>(stream)), "gdn_conv launch");
}

int gdn_conv_pool(const void* x, int64_t x_batch_stride, int64_t x_row_stride, const void* weight,
                  const void* bias, void* state_pool, int64_t pool_size, const int32_t* in_slots,
                  const int32_t* out_slots, void* const* outputs, const int64_t* widths, int num_outputs,
                  int64_t B, int64_t T, int64_t D, int64_t W, int dtype, int flags, void* stream) {
  gdn::ConvArgs a{};
  if (B < 0) return fail(GDN_ERR_VALUE, "batch_size must be non-negative");
  if (T < 1) return fail(GDN_ERR_VALUE, "seq_len must be at least 1");
  if (pool_size < 0 || pool_size > INT32_MAX)
    return fail(GDN_ERR_VALUE, "pool_size must be non-negative and fit int32 slot indices");
  if (B == 0) return ok();
  if (int e = check_conv(x, x_batch_stride, x_row_stride, weight, bias, outputs, widths, num_outputs, T, B,
                         D, W, dtype, flags, &a))
    return e;
  if (!in_slots || (pool_size > 0 && !state_pool)) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(state_pool, 16)) return fail(GDN_ERR_VALUE, "state_pool must be 16-byte aligned");
  if (!aligned(in_slots, 4) || !aligned(out_slots, 4))
    return fail(GDN_ERR_VALUE, "slot arrays must be 4-byte aligned");
  if (conv_overlap(a, B * T, (B - 1) * x_batch_stride + (T - 1) * x_row_stride + D,
                   {state_pool, static_cast<size_t>(pool_size) * (W - 1) * D * 2}, nullptr))
    return fail(GDN_ERR_VALUE, "an output overlaps another tensor");
  a.pool = state_pool;
  a.pool_size = pool_size;
  a.in_slots = in_slots;
  a.out_slots = out_slots;
  return cuda_status(gdn::launch_conv(a, static_cast<cudaStream_t>(stream)), "gdn_conv_pool launch");
}

static int check_ssm(const void* x, const void* B, const void* C, const float* A_log, const void* a,
                     const float* dt_bias, const void* y, int64_t T, int64_t H, int64_t G, int64_t P,
                     int64_t Ns) {
  if (H <= 0 || G <= 0 || H % G != 0)
    return fail(GDN_ERR_VALUE, "num_heads (%lld) must be a positive multiple of num_groups (%lld)",
                (long long)H, (long long)G);
  if (H > 65536) return fail(GDN_ERR_VALUE, "num_heads must be at most 65536 (got %lld)", (long long)H);
  if (P != 64 && P != 128) return fail(GDN_ERR_VALUE, "head_dim must be 64 or 128 (got %lld)", (long long)P);
  if (Ns != 64 && Ns != 128)
    return fail(GDN_ERR_VALUE, "state_dim must be 64 or 128 (got %lld)", (long long)Ns);
  if (!A_log || !dt_bias || (T > 0 && (!x || !B || !C || !a || !y)))
    return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(x, 16) || !aligned(B, 16) || !aligned(C, 16) || !aligned(y, 16) || !aligned(a, 2))
    return fail(GDN_ERR_VALUE, "x, B, C and output must be 16-byte aligned");
  return GDN_OK;
}

// Token by token for means of up to 16 tokens a sequence: measured with 1 to 32 sequences of 8 to 64
// heads the kernels cross between 12 and 24 tokens (one sequence, 64 heads: 8.0 against 9.3 us at
// 16 tokens, 10.4 against 9.4 at 24; 32 sequences: 45 against 66 us at 8, 70 against 67 at 16).
// Only the mean is known on the host, and one long sequence among short ones walks all its tokens
// (0.3 us each): the second bound holds what such a call can lose to about the chunked kernel's time.
static bool ssm_recurrent(int64_t T, int64_t N, int64_t H, int64_t G, int64_t P) {
  const int64_t tiles = G * ((H / G * P + 127) / 128);
  return T <= 16 * N && 2 * T <= (N * tiles > 128 ? N * tiles : 128);
}

// The scan's outputs against its inputs, `rows` tokens and states of `bytes` bytes.  (A call in two
// launches reads x and a in the first while the second writes.)
static bool ssm_overlap(const gdn::SsmArgs& p, int64_t rows, const void* states, const void* new_states, size_t bytes,
                        Range workspace) {
  const size_t x = static_cast<size_t>(rows) * p.H * p.P * 2, b = static_cast<size_t>(rows) * p.G * p.Ns * 2,
               heads = static_cast<size_t>(p.H) * 4;
  const Range w[3] = {{p.out, x}, {new_states, bytes}, workspace};
  const Range r[8] = {{p.x, x}, {p.B, b}, {p.C, b}, {p.a, static_cast<size_t>(rows) * p.H * 2}, {states, bytes},
                      {p.A_log, heads}, {p.dt_bias, heads}, {p.D, heads}};
  return any_overlap(w, 3, r, 8);
}

size_t gdn_ssm_workspace_bytes(int64_t T, int64_t N, int64_t H, int64_t G, int64_t P, int64_t Ns) {
  if (T <= 0 || N <= 0 || T > 0x7fffffffLL - 64 || N > 0x7fffffffLL || H > 65536 || H <= 0 || G <= 0 || H % G != 0 || (P != 64 && P != 128) || (Ns != 64 && Ns != 128) ||
      ssm_recurrent(T, N, H, G, P))
    return 0;
  return gdn::ssm_chunked_workspace(T, N, H, G, P, Ns, sm_count());
}

int gdn_ssm(const void* x, const void* B, const void* C, const float* state, const float* A_log,
            const void* a, const float* dt_bias, const float* D, const int64_t* cu_seqlens, void* output,
            float* new_state, int64_t T, int64_t N, int64_t H, int64_t G, int64_t P, int64_t Ns,
            void* workspace, size_t workspace_bytes, void* stream) {
  if (N <= 0) return fail(GDN_ERR_VALUE, "must have at least one sequence");
  if (T < 0) return fail(GDN_ERR_VALUE, "total_seq_len must be non-negative");
  if (int e = check_ssm(x, B, C, A_log, a, dt_bias, output, T, H, G, P, Ns)) return e;
  if (!cu_seqlens || !new_state) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(state, 16) || !aligned(new_state, 16) || !aligned(cu_seqlens, 8))
    return fail(GDN_ERR_VALUE, "state and new_state must be 16-byte and cu_seqlens 8-byte aligned");
  if (T > 0x7fffffffLL - 64) return fail(GDN_ERR_VALUE, "total_seq_len too large");
  if (N > 0x7fffffffLL / (H * P)) return fail(GDN_ERR_VALUE, "too many state rows (num_seqs x num_heads x head_dim)");
  const size_t bytes = static_cast<size_t>(N) * H * P * Ns * 4;
  if (overlap(state, bytes, new_state, bytes)) return fail(GDN_ERR_VALUE, "new_state overlaps state");
  const size_t need = gdn_ssm_workspace_bytes(T, N, H, G, P, Ns);
  if (workspace && workspace_bytes < need) return fail(GDN_ERR_VALUE, "workspace needs %zu bytes", need);
  if (!aligned(workspace, 256)) return fail(GDN_ERR_VALUE, "workspace must be 256-byte aligned");
  gdn::SsmArgs p{};
  p.x = x, p.B = B, p.C = C, p.state = state, p.A_log = A_log, p.a = a, p.dt_bias = dt_bias, p.D = D;
  p.cu_seqlens = cu_seqlens, p.out = output, p.new_state = new_state;
  p.T = T, p.N = N, p.H = H, p.G = G, p.P = P, p.Ns = Ns;
  if (ssm_overlap(p, T, state, new_state, bytes, {workspace, need})) return fail(GDN_ERR_VALUE, "an output overlaps another tensor");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (ssm_recurrent(T, N, H, G, P)) return cuda_status(gdn::launch_ssm_recurrent(p, st), "gdn_ssm launch");
  return cuda_status(gdn::launch_ssm_chunked(p, need ? workspace : nullptr, sm_count(), st), "gdn_ssm launch");
}

int gdn_ssm_pool(const void* x, const void* B, const void* C, const float* A_log, const void* a,
                 const float* dt_bias, const float* D, void* state_pool, int state_dtype, int64_t pool_size,
                 const int32_t* in_slots, const int32_t* out_slots, int flags, void* output, int64_t batch,
                 int64_t T, int64_t H, int64_t G, int64_t P, int64_t Ns, void* stream) {
  if (batch < 0) return fail(GDN_ERR_VALUE, "batch_size must be non-negative");
  if (T < 1) return fail(GDN_ERR_VALUE, "seq_len must be at least 1");
  if (pool_size < 0 || pool_size > INT32_MAX)
    return fail(GDN_ERR_VALUE, "pool_size must be non-negative and fit int32 slot indices");
  if (state_dtype != GDN_STATE_F32 && state_dtype != GDN_STATE_BF16)
    return fail(GDN_ERR_TYPE, "state_dtype must be GDN_STATE_F32 or GDN_STATE_BF16");
  if (flags & ~GDN_POOL_NO_STATE_UPDATE) return fail(GDN_ERR_VALUE, "unknown flags");
  if (batch == 0) return ok();
  if (int e = check_ssm(x, B, C, A_log, a, dt_bias, output, T, H, G, P, Ns)) return e;
  if (!in_slots || (pool_size > 0 && !state_pool)) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(state_pool, 16)) return fail(GDN_ERR_VALUE, "state_pool must be 16-byte aligned");
  if (!aligned(in_slots, 4) || !aligned(out_slots, 4))
    return fail(GDN_ERR_VALUE, "slot arrays must be 4-byte aligned");
  gdn::SsmArgs p{};
  p.x = x, p.B = B, p.C = C, p.A_log = A_log, p.a = a, p.dt_bias = dt_bias, p.D = D;
  p.out = output, p.pool = state_pool, p.in_slots = in_slots, p.out_slots = out_slots;
  p.T = T, p.N = batch, p.H = H, p.G = G, p.P = P, p.Ns = Ns, p.pool_size = pool_size;
  p.state_bf16 = state_dtype == GDN_STATE_BF16;
  p.no_state_update = (flags & GDN_POOL_NO_STATE_UPDATE) != 0;
  if (ssm_overlap(p, batch * T, nullptr, state_pool,
                  static_cast<size_t>(pool_size) * H * P * Ns * (p.state_bf16 ? 2 : 4), {nullptr, 0}))
    return fail(GDN_ERR_VALUE, "an output overlaps another tensor");
  return cuda_status(gdn::launch_ssm_recurrent(p, static_cast<cudaStream_t>(stream)), "gdn_ssm_pool launch");
}

int gdn_rms_norm(const void* x, int64_t x_stride, const void* weight, const void* residual,
                 int64_t residual_stride, const void* gate, int64_t gate_stride, float eps, void* output,
                 float* scale, int64_t group, void* residual_out, int64_t rows, int64_t D, int dtype,
                 int flags, void* stream) {
  if (D <= 0 || D % 8 != 0 || D > 16384)
    return fail(GDN_ERR_VALUE, "dim must be a multiple of 8 up to 16384 (got %lld)", (long long)D);
  if (rows < 0) return fail(GDN_ERR_VALUE, "rows must be non-negative");
  if (dtype != GDN_BF16 && dtype != GDN_F16) return fail(GDN_ERR_TYPE, "dtype must be GDN_BF16 or GDN_F16");
  if (flags & ~GDN_NORM_GATE_FIRST) return fail(GDN_ERR_VALUE, "unknown flags");
  if (group != 0 && (group != 128 || D % 128 != 0))
    return fail(GDN_ERR_VALUE, "group_size must be 0, or 128 with dim a multiple of 128");
  if (group != 0 && !scale) return fail(GDN_ERR_VALUE, "group_size needs a scale output");
  if (residual && gate) return fail(GDN_ERR_VALUE, "residual and gate cannot both be given");
  if ((residual != nullptr) != (residual_out != nullptr) && rows > 0)
    return fail(GDN_ERR_VALUE, "residual_out goes with residual");
  if (rows == 0) return ok();
  if (!x || !weight || !output) return fail(GDN_ERR_VALUE, "null pointer argument");
  if (!aligned(x, 16) || !aligned(weight, 16) || !aligned(residual, 16) || !aligned(gate, 16) ||
      !aligned(output, 16) || !aligned(residual_out, 16) || !aligned(scale, 4))
    return fail(GDN_ERR_VALUE, "buffers must be 16-byte aligned");
  const int64_t strides[3] = {x_stride, residual ? residual_stride : D, gate ? gate_stride : D};
  for (int64_t st : strides)
    if (st < D || st % 8 != 0)
      return fail(GDN_ERR_VALUE, "row strides must be multiples of 8 and at least dim");
  const size_t span = (static_cast<size_t>(rows - 1) * (residual ? residual_stride : D) + D) * 2;
  if (residual && overlap(residual, span, residual_out, static_cast<size_t>(rows) * D * 2) &&
      !(residual == residual_out && residual_stride == D))
    return fail(GDN_ERR_VALUE, "residual_out overlaps residual without being the same buffer");
  // a row may be replaced by its own result (a thread reads its values before it writes them), no other
  const size_t out_bytes = static_cast<size_t>(rows) * D * (scale ? 1 : 2), flat = static_cast<size_t>(rows) * D * 2;
  const Range in[3] = {{x, (static_cast<size_t>(rows - 1) * strides[0] + D) * 2}, {residual, span},
                       {gate, (static_cast<size_t>(rows - 1) * strides[2] + D) * 2}};
  for (int i = 0; i < 3; ++i) {
    const bool same = strides[i] == D;
    if ((overlap(output, out_bytes, in[i].p, in[i].bytes) && !(same && !scale && output == in[i].p)) ||
        (overlap(residual_out, flat, in[i].p, in[i].bytes) && !(same && residual_out == in[i].p)))
      return fail(GDN_ERR_VALUE, "an output overlaps an input without being the same buffer");
  }
  if (overlap(output, out_bytes, residual_out, flat)) return fail(GDN_ERR_VALUE, "output overlaps residual_out");
  // the scales and the weight share nothing
  const Range written[3] = {{output, out_bytes}, {residual_out, flat},
                            {scale, static_cast<size_t>(rows) * (group ? D / group : 1) * 4}};
  for (int i = 0; i < 3; ++i)
    if (overlap(weight, static_cast<size_t>(D) * 2, written[i].p, written[i].bytes) ||
        overlap(written[2].p, written[2].bytes, in[i].p, in[i].bytes) ||
        (i < 2 && overlap(written[2].p, written[2].bytes, written[i].p, written[i].bytes)))
      return fail(GDN_ERR_VALUE, "weight or scale overlaps another tensor");
  const gdn::NormArgs a{x, weight, residual, gate, output, scale, residual_out, x_stride, residual_stride,
                        gate_stride, rows, D, group, eps, dtype == GDN_F16,
                        (flags & GDN_NORM_GATE_FIRST) != 0};
  return cuda_status(gdn::launch_rms_norm(a, static_cast<cudaStream_t>(stream)), "gdn_rms_norm launch");
}

}  // extern "C"
