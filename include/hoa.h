/*
 * hoa.h — C ABI of the B200 (sm_100a) path-ordered geometric attention forward.
 *
 * The library (libhoa.so) implements the causal forward of
 * PathOrderedGeometricMHA from SiddhiMali/HolonomyAwareAttention between the
 * PyTorch projections: it takes the edge-MLP output a_all and the qkv
 * projection, and returns the per-head outputs that feed the `out` Linear.
 *
 *   G_t  = expm(skew(edge_scale * a_t))          t = 0 .. T-2   (edge t joins t, t+1)
 *   P_0  = I,  P_{t+1} = G_t P_t
 *   q^_t = P_t^T q_t,  k^_t = P_t^T k_t,  v^_t = P_t^T v_t
 *   o_i  = P_i * sum_{j<=i} softmax_j(q^_i . k^_j * softmax_scale) v^_j
 *
 * Layout conventions (row-major, contiguous):
 *   a_all  (B, T, H, m)    m = d(d-1)/2, row-major strict upper triangle per head
 *   qkv    (B, T, H, 3d)   per head [q | k | v]  (the reference's qkv(x).view(B,T,H,3d))
 *   out    (B, T, H, d)    i.e. the (B, T, D) input of the `out` projection
 *   chain c = b*H + h.  Rotations are always fp32.
 *
 * Rules of the ABI: no entry point allocates or synchronises; all work is
 * enqueued on the caller's stream (`stream` is a cudaStream_t, NULL = legacy
 * default stream).  Scratch comes from the caller through `workspace`
 * (hoa_core_workspace_bytes).  Every entry point returns a hoa_status.
 *
 * Process-wide state (everything else keeps none, and may be called from
 * several host threads on different data):
 *   - hoa_edge_gemm and hoa_edge_gemm_fp8_acc keep one cuBLASLt handle and a
 *     plan per GEMM shape, and serialise their calls with a lock;
 *   - hoa_core_forward_noalloc computes in one static device array per GPU,
 *     shared by all its calls (see there), and caches that array's address
 *     per device;
 *   - hoa_set_wait_bound sets the bound of the device-side waits of every
 *     kernel launched after it (a diagnostic; the default is seconds).
 * The generation entry points ask the driver once per device for their kernels'
 * shared memory, and their kernels may come up while the one before them in the
 * stream drains; each waits for all work before it before it touches memory.
 * Kernels whose bounded waits can give up report HOA_ERR_TIMEOUT through a
 * device status word (hoa_core_forward: the first 4 bytes of the workspace;
 * the stage entry points: their `status` argument).  The status of a launch is
 * known only once its stream has completed: read the word then.
 */
#ifndef HOA_H_
#define HOA_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  HOA_OK = 0,
  HOA_ERR_INVALID_ARG = 1,   /* null pointer, bad shape, misaligned pointer */
  HOA_ERR_UNSUPPORTED = 2,   /* head dim or dtype outside the compiled set  */
  HOA_ERR_LAUNCH = 3,        /* CUDA launch failed (cudaGetLastError)       */
  HOA_ERR_WORKSPACE = 4,     /* workspace too small                          */
  HOA_ERR_TIMEOUT = 5,       /* a bounded device-side wait gave up           */
  HOA_ERR_BOUNDS = 6,        /* debug build: a device-side index check failed */
  HOA_ERR_PAGES = 7          /* cache: no free page, or a row or page outside it */
} hoa_status;

typedef enum { HOA_F32 = 0, HOA_BF16 = 1 } hoa_dtype;

/*
 * Generator layout flag, OR'ed into `a_dtype` (with HOA_F32 only, for head
 * dims d % 32 == 0).  Without it the d(d-1)/2 generators of a head are packed
 * as the reference packs them: the strict upper triangle row by row
 * (core/utils.py skew_from_vec; entry (i, j), i < j, at i(2d-i-1)/2 + j-i-1).
 * With it each head holds hoa_gen_stride(d, 1) floats and entry {i, j} sits at
 * slot 32k + ((i + j) mod 32): a permutation of the same values (plus a few
 * unused slots) chosen so that the link kernel reads each row of the skew
 * matrix from shared memory without bank conflicts.  A caller gets this layout
 * for free by permuting the output rows of the generator projection once
 * (hoa_gen_banked_map).  Both layouts give bit-identical results.
 */
#define HOA_GEN_BANKED 0x100

/* Library facts. */
int hoa_abi_version(void);
int hoa_max_head_dim(void);
const char* hoa_status_string(int status);

/* Chunk length used to split each (b,h) rotation chain into independent
 * chunks (composed locally, then joined by hoa_carry_scan).  `num_sms` is the
 * device's SM count.  Returns a length in [16, T] (T when T < 16) chosen so
 * that the link kernel's (chain, chunk) units fill whole waves of the GPU. */
int hoa_plan_chunk(int B, int H, int T, int d, int num_sms);

/*
 * The edge MLP's hidden layer as the bf16 operand of hoa_edge_gemm:
 * g = GELU(h) (exact erf, nn.GELU(); core/attention_fast_chunked.py:56-58) for
 * h (rows, cols) fp32, written as out (rows, cols) = bf16(g), or with split
 * (rows, 2 cols) = [bf16(g) | bf16(g - bf16(g))].  cols % 4 == 0, h 16-byte
 * aligned.  No reference counterpart beyond the GELU itself.
 */
int hoa_edge_gelu_split(const float* h, void* out, long long rows, int cols, int split, void* stream);

/* Floats per head of the generator row: d(d-1)/2 (banked = 0) or the banked
 * layout's size (banked = 1; 0 when d % 32 != 0). */
int hoa_gen_stride(int d, int banked);

/* slot_of_index[i] (i < d(d-1)/2, reference order) = the banked slot of
 * reference entry i.  Returns HOA_ERR_UNSUPPORTED when d % 32 != 0. */
int hoa_gen_banked_map(int d, int* slot_of_index);

/* Bytes of scratch hoa_core_forward needs.  The first 4 bytes of the
 * workspace receive a device status word (0, or HOA_ERR_TIMEOUT when a
 * bounded device-side wait gave up); read it after the stream completes. */
size_t hoa_core_workspace_bytes(int B, int H, int T, int d, int chunk, int hat_dtype);

/*
 * Whole core region in one call: kernels (1)-(4).
 * Replaces the reference's core region between the projections:
 *   core/attention_fast_chunked.py:86-95   so_exp(skew_from_vec(a)) + prefix loop
 *   core/attention_fast_chunked.py:108-110 transport q^, k^, v^
 *   core/attention_fast_chunked.py:119-171 causal fold and out_i = P_i o_i
 * (kernel/attention_kernel.py:215-216 `_geometry` + `HoloAttnFn.apply`).
 * a_dtype / qkv_dtype / out_dtype: HOA_F32 or HOA_BF16.  `a_bias` (nullable,
 * (H*m) fp32) is added to every generator before the edge_scale multiply — the
 * edge MLP's output bias, so that the projection GEMM may leave it out
 * (core/attention_fast_chunked.py:76-77).  hat_dtype is the
 * dtype of the transported q^/k^/v^ fed to attention: HOA_BF16 runs the
 * tcgen05 tensor-core attention (d % 8 == 0, d <= 128), HOA_F32 the fp32 SIMT
 * attention.  `carry_in` (nullable, (B*H, d, d) fp32) is P at the first
 * position (a previous shard's product; NULL = identity); `total_out`
 * (nullable, (B*H, d, d)) receives the product through the last edge
 * t = T-1 (for a full sequence that edge is the closing edge, and total_out
 * is the holonomy G_close P_{T-1}, core/attention_fast_chunked.py:95).
 */
int hoa_core_forward(const void* a_all, int a_dtype, const float* a_bias, float edge_scale,
                     const void* qkv, int qkv_dtype,
                     void* out, int out_dtype, int hat_dtype, float softmax_scale,
                     const float* carry_in, float* total_out,
                     int B, int H, int T, int d, int chunk,
                     void* workspace, size_t workspace_bytes, void* stream);

/*
 * Kernels (1)+(2), local part: per (chain, chunk) unit, builds
 * G_t = expm(skew(edge_scale*a_t)) in fp32 and the local products
 * R_{t0} = I, R_{t+1} = G_t R_t over the chunk's edges.
 * Writes R (B*H, T, d, d) fp32 — R_t for every position —, the locally
 * transported vectors U (B*H, T, 3, d) fp32 = R_t^T [q_t, k_t, v_t], and the
 * chunk totals M (B*H, K, d, d) = R after the chunk's last edge.
 * `status` (nullable device int) receives HOA_ERR_TIMEOUT if a bounded
 * device-side wait gave up (the word is only ever set, never cleared).
 * Replaces core/attention_fast_chunked.py:86-94 (with core/utils.py:4-52)
 * and the transport at :108-110, split into independent chunks.
 */
int hoa_link_local(const void* a_all, int a_dtype, const float* a_bias, float edge_scale,
                   const void* qkv, int qkv_dtype,
                   float* R, float* U, float* M, int* status,
                   int B, int H, int T, int d, int chunk, void* stream);

/*
 * Kernel (2), carry: C_0 = carry_in (or I), C_{k+1} = M_k C_k for the K
 * chunks of each chain; writes C (B*H, K, d, d) and, if total_out != NULL,
 * C_K.  Joins the chunks so that P_t = R_t C_{t/chunk}
 * (core/attention_fast_chunked.py:91-94 re-associated).
 */
int hoa_carry_scan(const float* M, const float* carry_in, float* C, float* total_out,
                   int BH, int K, int d, void* stream);

/*
 * Kernel (2), transport: q^_t = C_k^T U_q[t] (likewise k, v) in hat_dtype.
 * q^, k^: (B*H, T, d).  v^: (B*H, T, d) when vt_stride == 0, else transposed
 * as (B*H, d, vt_stride) with vt_stride = hoa_vt_stride(T) (the layout
 * hoa_attn_tc_fwd reads).  Completes core/attention_fast_chunked.py:108-110.
 */
int hoa_carry_apply(const float* U, const float* C, void* qh, void* kh, void* vh,
                    int hat_dtype, int vt_stride, int BH, int T, int d, int chunk,
                    void* stream);

/* Row stride (elements) of the transposed v^ buffer: T rounded up to 8. */
int hoa_vt_stride(int T);

/*
 * Kernel (3), fp32 path: causal online-softmax attention with every product
 * in fp32.  q^ is (B*H, Tq, d), k^ and v^ (B*H, Tk, d), in fp32 (or bf16).
 * Query row i is global position q_offset + i and attends to keys
 * 0 .. q_offset + i (q_offset + Tq <= Tk; a whole sequence is Tq = Tk,
 * q_offset = 0; a sequence shard passes its offset and the gathered keys).
 * Writes the normalised o = softmax(q^ k^T * scale) v^ as (B*H, Tq, d) fp32.
 * Replaces core/attention_fast_chunked.py:119-168 (kernel/attention_kernel.py:122-134
 * run_fwd_kernel) for the causal tril mask.
 */
int hoa_attn_fwd(const void* qh, const void* kh, const void* vh, int hat_dtype,
                 float* o, float softmax_scale, int BH, int Tq, int Tk, int q_offset,
                 int d, void* stream);

/*
 * Kernel (3), bf16 path on tcgen05/TMEM: same contract as hoa_attn_fwd with
 * bf16 q^ (B*H, Tq, d), k^ (B*H, Tk, d) and v^ transposed
 * (B*H, d, hoa_vt_stride(Tk)); fp32 accumulation.  d % 8 == 0, d <= 128.
 * `status` (nullable device int) receives HOA_ERR_TIMEOUT if a bounded wait
 * gave up.
 */
int hoa_attn_tc_fwd(const void* qh, const void* kh, const void* vhT, float* o, int* status,
                    float softmax_scale, int BH, int Tq, int Tk, int q_offset, int d,
                    void* stream);

/*
 * The path products P_t = R_t C_{t/chunk} (B*H, T, d, d) in p_dtype, from the
 * link kernel's R and the carry scan's C: the "C" entry of the reference's
 * forward(..., return_geometry=True) (core/attention_fast_chunked.py:89-94,
 * 175-177; its "H" entry, the holonomy, is hoa_carry_scan's total_out).  Not on
 * the forward's path, which never materialises P.
 */
int hoa_compose_paths(const float* R, const float* C, void* P, int p_dtype, int BH, int T, int d,
                      int chunk, void* stream);

/*
 * General forms of the module (core/attention.py:69-195) beside the causal
 * tril path, all fp32, (B*H, T, d) row-major vectors:
 *
 * hoa_attn_general_fwd — softmax over all keys of a chain: o_i =
 *   sum_j softmax_j(q^_i . key_ij * scale) value_ij / l.clamp_min(1e-20), with
 *   key/value_ij = k^_j / v^_j for j <= i and, when kw/vw are given (both or
 *   neither), kw_j / vw_j for the wrap pairs j > i (the arc transport through
 *   the closing edge, core/attention.py:156-165: kw = Hol k^, vw = Hol v^).
 *   mask: (T, T) bytes, nonzero = allowed, NULL = all allowed; masked scores
 *   sit at -FLT_MAX as the reference's finfo.min (a fully masked row averages
 *   uniformly, core/attention_fast_chunked.py:142-148).  d <= 128.
 * hoa_chain_matvec — y_t = M x_t (transpose = 0) or M^T x_t, M (B*H, d, d).
 * hoa_apply_paths — y_t = P_t x_t (transpose = 0) or P_t^T x_t with
 *   P_t = R_t C_{t/chunk} (the inert ablation's transports,
 *   core/attention.py:166-169).
 */
int hoa_attn_general_fwd(const float* qh, const float* kh, const float* vh, const float* kw,
                         const float* vw, const unsigned char* mask, float* o, float softmax_scale,
                         int BH, int T, int d, void* stream);
int hoa_chain_matvec(const float* x, const float* M, float* y, int transpose, int BH, int T, int d,
                     void* stream);
int hoa_apply_paths(const float* x, const float* R, const float* C, int chunk, float* y, int transpose,
                    int BH, int T, int d, void* stream);

/*
 * Kernel (4): inverse transport out_t = R_t (C_{t/chunk} o_t), written to
 * out (B, T, H, d) in out_dtype — the input of the `out` projection.
 * Replaces core/attention_fast_chunked.py:171.
 */
int hoa_out_transport(const float* o, const float* R, const float* C, int chunk,
                      void* out, int out_dtype, int B, int H, int T, int d, void* stream);

/* Size of the static scratch behind hoa_core_forward_noalloc: 16 MiB. */
#define HOA_NOALLOC_SCRATCH_BYTES (16u * 1024u * 1024u)

/*
 * hoa_core_forward_noalloc — no counterpart in the reference.  Same
 * computation and arguments as hoa_core_forward minus the workspace, for
 * callers that cannot allocate device memory when they call in (for example
 * an inference-engine plugin whose enqueue callback must not call cudaMalloc,
 * or a process whose device memory is reserved in full by another allocator).
 * Its scratch is a static device array of HOA_NOALLOC_SCRATCH_BYTES inside
 * the library, which every GPU that loads it keeps until the process exits;
 * nothing is allocated per call.  Problems whose hoa_core_workspace_bytes
 * exceeds that size return HOA_ERR_WORKSPACE without enqueuing work.
 * It runs on the current device, and `stream` must belong to that device.
 * The first call on each device (and the first after a device reset, which
 * gives the device a new context) looks up the array's device address
 * (cudaGetSymbolAddress) and caches it, so make that first call before any
 * stream capture.  All calls share the array and it keeps the last call's
 * contents: calls that overlap on the GPU (other streams, other host
 * threads) race on it, so serialise them.  The call's device status word
 * (0, or HOA_ERR_TIMEOUT when a bounded device-side wait gave up) is cleared
 * at the start of every call and lies in the array: hoa_noalloc_status_word.
 */
int hoa_core_forward_noalloc(const void* a_all, int a_dtype, const float* a_bias,
                             float edge_scale,
                             const void* qkv, int qkv_dtype,
                             void* out, int out_dtype, int hat_dtype, float softmax_scale,
                             const float* carry_in, float* total_out,
                             int B, int H, int T, int d, int chunk, void* stream);

/*
 * hoa_noalloc_status_word — no counterpart in the reference.  The device
 * address, on the current device, of the status word that the last
 * hoa_core_forward_noalloc call on that device wrote: read it (4 bytes, e.g.
 * with cudaMemcpy) once that call's stream has completed.  Allocates nothing;
 * like hoa_core_forward_noalloc, its first call on a device does the address
 * look-up, so make it before any stream capture.
 */
int hoa_noalloc_status_word(int** dev_status);

/*
 * hoa_set_wait_bound — no counterpart in the reference.  A diagnostic: the
 * bound, in SM cycles, of the device-side waits (on TMA and tensor-core
 * completion) of every kernel launched after the call, process-wide.
 * 0 restores the default (4e9 cycles, i.e. seconds); the maximum is the
 * default.  A short bound makes a real forward's waits give up: the kernels
 * then leave early without faulting (each waits, with the default bound, for
 * its copies and products in flight, frees its tensor memory and returns) and
 * report HOA_ERR_TIMEOUT in their status word; the output is not valid.
 */
int hoa_set_wait_bound(long long max_cycles);

/*
 * hoa_debug_bounds — no counterpart in the reference.  Device-side index
 * checks of the debug build (libhoa_debug.so, built with -DHOA_DEBUG_BOUNDS;
 * compute-sanitizer is not available where this library is tested).  In that
 * build every kernel of the core path checks, before each global access, that
 * the element range a unit (a position, a chunk, a row) touches lies inside
 * the extent its buffer has for the launch's shape; a check that fails
 * records HOA_ERR_BOUNDS and the access is skipped (never performed; a
 * skipped TMA copy completes its barrier with zero bytes), so nothing faults
 * or traps.  The call returns in *status (host int) the first code recorded
 * since the previous call on this device (0 if none) and clears it, after
 * waiting for the device to finish; it then sets every check to compare
 * against extents shifted right by `extent_shift` (0 = the true extents; a
 * test hook: 1 makes the checks treat every buffer as half as long, so they
 * fire on accesses that are really in bounds).  The product build returns
 * HOA_ERR_UNSUPPORTED.
 */
int hoa_debug_bounds(int extent_shift, int* status);

/*
 * hoa_edge_gemm — the second layer of the edge MLP (core/attention_fast_chunked.py:76,
 * `edge_mlp[2]`, whose output is the a_all of hoa_core_forward) as one cuBLASLt GEMM, a plain
 * library GEMM: out (M x N, fp32, row-major) = hidden (M x K, bf16, row-major) * wt (K x N,
 * bf16, row-major, i.e. W^T) + bias (N floats, nullable), fp32 accumulation, the bias added in
 * the GEMM's epilogue.  workspace: caller-owned cuBLASLt scratch (32 MiB is plenty).  The plan
 * of each shape is made once and cached; calls are serialised inside the library.
 */
int hoa_edge_gemm(const void* hidden, const void* wt, const float* bias, float* out, int M, int N,
                  int K, void* workspace, size_t workspace_bytes, void* stream);

/*
 * The low half of the edge MLP's second layer in fp8 (the same layer as hoa_edge_gemm,
 * core/attention_fast_chunked.py:76; the reference computes it in one fp32 GEMM): with
 * g = g_hi + g_lo, g_hi = bf16(g), the layer is W g_hi + W g_lo; the first term is a bf16
 * hoa_edge_gemm and the second, whose terms are at most 2^-9 of the first's, this call:
 *   hoa_edge_gelu_split8: g = GELU(h) (exact erf) for h (rows, cols) fp32 -> hi (rows, cols)
 *     = bf16(g) and lo (rows, cols) = e4m3(lo_scale * (g - bf16(g))), saturating (one byte
 *     each); cols % 4 == 0, h 16-byte aligned, lo_scale > 0 (a power of two keeps it exact);
 *   hoa_edge_gemm_fp8_acc: out (M x N, fp32, row-major) += alpha * lo (M x K, e4m3,
 *     row-major) * w^T, w (N x K, e4m3, row-major: the weight as nn.Linear stores it), fp32
 *     accumulation; alpha undoes the two operands' scales.  M, N, K multiples of 16.
 * The plan of each shape is made once and cached; calls are serialised inside the library.
 */
int hoa_edge_gelu_split8(const float* h, void* hi, void* lo, long long rows, int cols, float lo_scale,
                         void* stream);
int hoa_edge_gemm_fp8_acc(const void* lo, const void* w, float* out, float alpha, int M, int N, int K,
                          void* workspace, size_t workspace_bytes, void* stream);

/*
 * ---------------------------------------------------------------------------
 * Generation: pages of a cache, attention over them, and the path step of one
 * token.  No counterpart in the reference, which recomputes the whole sequence:
 * k^_t = P_t^T k_t and v^_t = P_t^T v_t are in the gauge of their sequence's
 * origin, so a token's k^ and v^ never change as the sequence grows, and
 * sequences with a common beginning share them.
 *
 * A pool holds pages (n_pages, H, page, d) of fp32 or bf16, innermost dimension
 * contiguous; k and v pools of a call have the same `page_strides` (elements:
 * page, head, token).  Bookkeeping is int32 on the device: table (S, W) the page
 * ids of each row in order, -1 beyond its last; lens (S) its tokens; refs
 * (n_pages) the rows that hold a page (0: free).  Row s uses ceil(lens[s] / page)
 * entries.  Page ids and rows read from device memory are checked by the kernels:
 * one outside the cache is not followed, and sets HOA_ERR_PAGES in `status`
 * (nullable; device or mapped host int, only ever set; known once the stream has
 * completed).
 * ---------------------------------------------------------------------------
 *
 * The bookkeeping entry points read one state and write the next one to other
 * buffers (same shapes), in one launch; free pages are taken lowest index first
 * and requests served in list order, so results are reproducible.
 *   reserve  row s grows by counts[s] tokens.
 *   fork     row dst[i] (empty) becomes a copy of row src[i], i < n: full pages
 *            are shared, a last page that is not full is copied in every pool.
 *   free     the rows end; pages that no row holds any more are free.
 *   compact  the *live pages move to 0 .. live-1 in every pool and the table
 *            follows, so that the pool's tail can be given up.
 * reserve and fork are all or nothing: with too few free pages or an invalid
 * request (a row outside the table, a dst that is not empty or listed twice, a
 * row longer than W pages or 2^31 - 1 tokens) the new state equals the old one, no payload moves,
 * and `status` is set.  S <= 65536, S * W < 2^31, and n and n_pages
 * at most 2^31 - 65536.
 * pools / strides / bytes: n_pools base pointers, bytes between pages and bytes
 * of a page; host arrays, read during the call.  Payload moves only into pages
 * that are free in the old state.
 *   hoa_pages_copy   page to[i] = page from[i] in every pool, i < n (device
 *            lists; both -1: skipped); no page is both read and written.
 *   hoa_pages_write  k, v (B, T, H, d) (strides of row, token, head) become the
 *            last T tokens of each row: token t goes to position lens[b] - T + t
 *            (not written where that is negative).
 */
size_t hoa_pages_workspace_bytes(int n, int n_pages);
int hoa_pages_reserve(const int* table, const int* lens, const int* refs, const int* counts, int* table_out,
                      int* lens_out, int* refs_out, int S, int W, int n_pages, int page, void* workspace,
                      size_t workspace_bytes, int* status, void* stream);
int hoa_pages_fork(const int* table, const int* lens, const int* refs, const int* src, const int* dst, int n,
                   int* table_out, int* lens_out, int* refs_out, int S, int W, int n_pages, int page,
                   void* const* pools, const long long* strides, const long long* bytes, int n_pools,
                   void* workspace, size_t workspace_bytes, int* status, void* stream);
int hoa_pages_free(const int* table, const int* lens, const int* refs, const int* rows, int n, int* table_out,
                   int* lens_out, int* refs_out, int S, int W, int n_pages, int page, int* status, void* stream);
int hoa_pages_compact(const int* table, const int* refs, int* table_out, int* refs_out, int* live, int S, int W,
                      int n_pages, void* const* pools, const long long* strides, const long long* bytes, int n_pools,
                      void* workspace, size_t workspace_bytes, int* status, void* stream);
int hoa_pages_copy(void* const* pools, const long long* strides, const long long* bytes, int n_pools,
                   const int* from, const int* to, int n, int n_pages, int* status, void* stream);
int hoa_pages_write(const void* k, const void* v, int src_dtype, const long long* k_strides,
                    const long long* v_strides, void* k_pages, void* v_pages, int dtype,
                    const long long* page_strides, const int* table, long long table_stride, const int* lens,
                    int B, int T, int H, int d, int page, int W, int n_pages, int* status, void* stream);

/*
 * Attention of B rows over the cache.  q (B, Tq, H, d) (strides of row, token,
 * head), H a multiple of the pools' Hk heads: query head h reads kv head
 * h / (H / Hk).  The first n_shared pages of every row are `shared` (their keys
 * are read once for the whole batch); `table` (B, W) holds the pages after them.
 * lens[b] counts all keys of row b, the shared ones and its Tq newest included:
 * query t sees keys 0 .. lens[b] - Tq + t.  A row may end inside the shared
 * pages, have fewer keys than queries, or none.
 *   out (B, Tq, H, d) = softmax(q k^T * scale) v, 0 where a query sees no key;
 *   lse (B, Tq, H) = the log of the softmax's sum, -inf there.
 * paths (nullable, Tq = 1): (B, H, d, d) fp32, then out = P o, the inverse
 * transport (core/attention_fast_chunked.py:171); a row that sees no key gives 0
 * whatever its P holds.  q and the pools share `dtype`;
 * d <= 128; B * Tq * H and (n_shared + W) * page at most 2^31 - 65536.
 * Slots that no query sees may hold anything, NaN included; a NaN or a
 * score of +inf that a query sees makes its out and lse NaN.  (A NaN or infinity in
 * v also reaches, as 0 times it, queries that do not see it but share a tile of keys
 * and rows with one that does.)  The workspace is
 * 16-byte aligned; calls that may overlap on the GPU use different ones.
 */
size_t hoa_paged_attn_workspace_bytes(int B, int Tq, int H, int Hk, int d, int page, int n_shared, int W, int num_sms);
int hoa_paged_attn_fwd(const void* q, const long long* q_strides, const void* k_pages, const void* v_pages,
                       const long long* page_strides, int dtype, const int* shared, int n_shared,
                       const int* table, long long table_stride, int W, const int* lens, const float* paths,
                       void* out, int out_dtype, float* lse, float softmax_scale, int B, int Tq, int H, int Hk,
                       int d, int page, int n_pages, int num_sms, void* workspace, size_t workspace_bytes,
                       int* status, void* stream);

/*
 * One generated token of every row: kernels (1) and (2) in their single-token form
 * (core/attention_fast_chunked.py:86-94, 108-110).
 *   P_out = expm(skew(edge_scale * (a + a_bias))) P     (B, H, d, d) fp32
 *   q^ = P_out^T q -> qh (B, H, d); k^, v^ likewise -> slot lens[b] - 1 of the row
 * a (B, H * stride) fp32: the generators of the edge from the row's previous token
 * to this one (a_dtype HOA_F32, with or without HOA_GEN_BANKED); qkv (B, H, 3d)
 * rows `qkv_stride` elements apart.  lens[b] counts the token itself: at lens 1
 * there is no edge and P_out = I; at lens 0 P_out = P, q^ = 0 and nothing is
 * written.  P_out may be P.  qh and the pools share `dtype`; 2 <= d <= 120,
 * B * H at most 2^31 - 65536.
 * The products run on the tensor cores in fixed-point ranges: entries of P are
 * those of a rotation (at most 1; up to 255 stay exact to 2^-22), and
 * |edge_scale * (a + a_bias)| < 4094.  `status` may also receive HOA_ERR_TIMEOUT.
 */
int hoa_path_step(const float* a, int a_dtype, const float* a_bias, float edge_scale, const float* P, float* P_out,
                  const void* qkv, int qkv_dtype, long long qkv_stride, void* qh, void* k_pages, void* v_pages,
                  int dtype, const long long* page_strides, const int* table, long long table_stride, int W,
                  const int* lens, int B, int H, int d, int page, int n_pages, int* status, void* stream);

/*
 * Training: the backward passes of kernels (1)-(4) and the optimizer's step.  (The reference
 * differentiates core/attention_fast_chunked.py:63-177 with autograd; kernel/attention_kernel.py:166-187
 * recomputes the forward.)
 *
 * hoa_attn_fwd_lse - hoa_attn_fwd that also leaves lse (B*H, Tq) fp32, the log-sum-exp of a row's scaled
 * scores, which the backward pass recomputes the probabilities from; v^ row-major.  bf16 with d % 8 == 0
 * runs on tcgen05, the rest in fp32 on the CUDA cores; d <= 128.  softmax_scale is positive and finite, here
 * and in hoa_attn_bwd.
 */
int hoa_attn_fwd_lse(const void* qh, const void* kh, const void* vh, int dtype, float* o, float* lse,
                     float softmax_scale, int BH, int Tq, int Tk, int q_offset, int d, int* status, void* stream);

/*
 * hoa_attn_bwd - gradients of causal attention (hoa_attn_fwd_lse) for the gradient `dout` (B*H, Tq, d) of o:
 *   p_ij = exp(scale q^_i.k^_j - lse_i) (j <= q_offset + i),  ds_ij = p_ij (dout_i.v^_j - dout_i.o_i)
 *   dq_i = scale sum_j ds_ij k^_j,  dk_j = scale sum_i ds_ij q^_i,  dv_j = sum_i p_ij dout_i
 * q^, k^, v^, dout and the three outputs are `dtype`, o and lse fp32; every output is written in full
 * (keys that no query sees: 0) and shares no memory with what is read.  Sums have a fixed order: two calls
 * give the same bits.  p and ds are fp32, in bf16 calls hi + lo to 2^-16 as operands; sums are fp32.  A NaN or
 * infinity in a position's k^ or v^ may also reach, as 0 times it, queries that do not see it, and one in a
 * query's q^, dout, o or lse keys that it does not see (in its tile of 64).  d <= 128,
 * B*H <= 65535.  The workspace is 256-byte aligned; `aligned`: q^, k^, v^, dout and the outputs all start at
 * 16-byte boundaries (bf16 otherwise, and with d % 8 != 0, goes through copies).  `status` may receive
 * HOA_ERR_TIMEOUT.
 */
size_t hoa_attn_bwd_workspace_bytes(int BH, int Tq, int Tk, int d, int dtype, int aligned);
int hoa_attn_bwd(const void* qh, const void* kh, const void* vh, const float* o, const float* lse, const void* dout,
                 int dtype, void* dq, void* dk, void* dv, float softmax_scale, int BH, int Tq, int Tk, int q_offset,
                 int d, void* workspace, size_t workspace_bytes, int* status, void* stream);

/*
 * hoa_path_bwd - gradients through the path P_t = R_t C_{t/chunk} (hoa_link_local, hoa_carry_scan) for those
 * of the attention's inputs (dq^, dk^, dv^: hoa_attn_bwd) and of its output o, doh = P^T dout
 * (hoa_apply_paths): da (B, T, H*stride) fp32 of the raw generators (in a_all's layout, unused slots 0; the
 * closing edge t = T - 1 gets 0) and dqkv (B, T, H, 3d) in out_dtype, [P dq^ | P dk^ | P dv^] a head.
 *   Z_t = sum_{s>t} skew(q^ dq^T + k^ dk^T + v^ dv^T + doh o^T)_s,  W = P_t Z_t P_t^T,
 *   da_t = edge_scale (phi(ad_A) W)_{i<j},  A = skew(edge_scale (a + a_bias)_t),  phi(z) = (e^z - 1)/z
 * q^, k^, v^, dq^, dk^, dv^, doh (B*H, T, d) are hat_dtype, o and everything between fp32.  P is taken as
 * orthogonal.  A position whose bound 2 min(||A||_inf, ||A||_F / sqrt 2) passes 480, or whose sums are not
 * finite, gets NaN.  2 <= d <= 120.  The workspace is 256-byte aligned.
 */
size_t hoa_path_bwd_workspace_bytes(int B, int H, int T, int d, int chunk);
int hoa_path_bwd(const float* a_all, int a_dtype, const float* a_bias, float edge_scale, const float* R, const float* C,
                 int chunk, const void* qh, const void* kh, const void* vh, const float* o, const void* dqh,
                 const void* dkh, const void* dvh, const void* doh, int hat_dtype, float* da, void* dqkv, int out_dtype,
                 int B, int H, int T, int d, void* workspace, size_t workspace_bytes, int* status, void* stream);

/*
 * hoa_adamw_step - one AdamW step over `count` tensors (host arrays of device pointers and of element
 * counts), in place, in one launch a 256 tensors:
 *   m = b1 m + (1-b1) g,  v = b2 v + (1-b2) g^2,  x = x (1 - lr wd) - lr/(1-b1^t) m / (sqrt(v)/sqrt(1-b2^t) + eps)
 * params p_dtype, grads g_dtype (each HOA_F32 or HOA_BF16).  masters (nullable, entries too): fp32 copies that the
 * step is made on; the parameter is then the copy, rounded.  What is written shares no memory with anything else that a
 * call is given (an fp32 parameter may be its own master).  state_bits 32: m and v fp32.  8: m and sqrt(v)
 * as e4m3 bytes, blocks of 256 elements, scales[i] (2, blocks) fp32: value = byte * scale, for m and for
 * sqrt(v).  step: device int32, the number t of this step, from 1.  The bytes are rounded to the nearest for beta1 up to
 * 15/16 and beta2 up to 0.95 (m towards 0 below 2^-5 of its scale where the gradient adds less than half of the smallest
 * step), else up or down by a hash of the element's number and t, so that the mean is exact.  A moment that is not finite
 * is held as NaN and is no part of its block's scale.
 */
int hoa_adamw_step(void* const* params, int p_dtype, float* const* masters, const void* const* grads, int g_dtype,
                   void* const* m, void* const* v, float* const* scales, int state_bits, const long long* sizes, int count,
                   const int* step, double lr, double beta1, double beta2, double eps, double weight_decay, void* stream);

/*
 * hoa_selftest_wait — no counterpart in the reference.  Diagnostic for the
 * bounded device-side waits every kernel of this library uses (mbarrier waits
 * on TMA and tensor-core completion): one CTA of two warps waits on two
 * mbarriers that nothing arrives at.  Warp 0 waits with a bound of max_cycles
 * SM cycles, gives up and raises the CTA's abort flag; warp 1 waits with the
 * library's full bound (seconds) but on the abort flag as well, so it must
 * give up as soon as warp 0 does.  Results, written to out[0..3] (device,
 * 4 ints): out[0] = HOA_ERR_TIMEOUT when warp 0 gave up, out[1] = 1 when
 * warp 1 left on the abort flag, out[2] = warp 1's wait in units of 1024
 * cycles, out[3] = 1 when both waits returned false.  Nothing faults or hangs:
 * the GPU context stays usable.  max_cycles must be in [1, 1e9].
 */
int hoa_selftest_wait(int* out, long long max_cycles, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HOA_H_ */
