/*
 * fsw.h — C ABI of the MI355X (gfx950) fused SwiGLU MLP forward.
 *
 * The reference (bit-ml/Fused-SwiGLU) has no C ABI: its internal boundary is the C++ template
 * `swiglu_fwd<TA,TB,TC>` declared at csrc/torch_bindings.cpp:16-27 and defined at
 * csrc/SwiGLU/swiglu.cu:397-525, plus the convenience op `fused_swiglu_bf16` (swiglu.cu:538-553).
 * The entry points below are what a foreign-function binding for that path binds instead; the
 * PyTorch operator surface (torch_bindings.cpp:31-50) is rebuilt on top of them.
 *
 * Conventions (all entry points):
 *   - every data pointer is a DEVICE pointer owned by the caller; nothing is allocated or freed here;
 *   - leading dimensions (ld*) are in ELEMENTS, inner (K) stride is 1 as in swiglu.cu:411-414;
 *   - `stream` is a hipStream_t passed as void* (NULL = the default stream); launches are
 *     asynchronous, nothing here synchronises;
 *   - the return value is FSW_OK (0) or a negative FSW_E_* code; nothing throws or aborts;
 *   - the fsw_validate_* functions touch no GPU API and can be called on a machine without one;
 *   - entry points are re-entrant: there is no process-wide mutable state apart from caches of device properties
 *     (filled atomically), so any number of host threads may call them on any streams at the same time;
 *   - the library links the HIP runtime (libamdhip64). A process must hold ONE copy of it: inside a PyTorch-ROCm
 *     process, load torch (which brings its own) BEFORE this library, or launches fail with FSW_E_DEVICE.
 *
 * Weight formats (identical to the reference's):
 *   W13 [N = 2*ff, K] row-major, K-contiguous, rows interleaved: row 2j   = "up"  (linear) operand,
 *                                                                row 2j+1 = "gate" (SiLU) operand
 *       (swiglu.cu:380-381, numeric_tests.py:41-43);
 *   W2  [D, FF] row-major, FF-contiguous (the transpose of the mathematical Wd[FF, D]).
 */
#ifndef FSW_H
#define FSW_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* every entry point below is exported; everything else in the library has hidden visibility */
#define FSW_API __attribute__((visibility("default")))

/* element types */
#define FSW_BF16 0
#define FSW_FP16 1

/* error codes */
#define FSW_OK            0
#define FSW_E_NULL       -1   /* a required pointer is NULL */
#define FSW_E_DTYPE      -2   /* dtype is not FSW_BF16 / FSW_FP16 */
#define FSW_E_SHAPE      -3   /* negative size, odd N, or a size beyond the supported range */
#define FSW_E_LD         -4   /* leading dimension smaller than the row it strides */
#define FSW_E_ALIGN      -5   /* K (or FF), a leading dimension or a pointer breaks the 16-byte rule */
#define FSW_E_WORKSPACE  -6   /* workspace missing or smaller than fsw_*_workspace_bytes() */
#define FSW_E_LAUNCH     -7   /* the HIP runtime rejected a launch (see fsw_last_hip_error) */
#define FSW_E_DEVICE     -8   /* the current device is not a gfx950 GPU */
#define FSW_E_VARIANT    -9   /* unknown kernel variant requested through fsw_set_variant */
#define FSW_E_STATIC_LIMIT -10 /* fsw_mlp_static: the shape needs more scratch than the library's static array */

/*
 * Host-only argument validation of fsw_gateup (replaces the dtype TORCH_CHECKs of swiglu.cu:475-480 and adds
 * the shape/stride checks the reference leaves out). Rules: M >= 0; N >= 0 and even; K >= 0 and K % 8 == 0
 * (16-byte vectors; the reference needs K % 32 == 0, swiglu.cu:220-230); ldx >= K, ldw >= K, ldh >= N/2;
 * ldx % 8 == 0 and ldw % 8 == 0; pointers non-NULL and X, W13 16-byte aligned when the problem is non-empty
 * (M == 0 or N == 0 needs no pointers; K == 0 needs only H, which is then written with zeros).
 */
FSW_API int fsw_validate_gateup(int dtype, int64_t M, int64_t N, int64_t K,
                        const void* X, int64_t ldx, const void* W13, int64_t ldw,
                        const void* H, int64_t ldh);

/*
 * H[M, N/2] = up * silu(gate) with up = X @ W13[0::2].T, gate = X @ W13[1::2].T; fp32 accumulation,
 * fp32 gating, ONE round-to-nearest-even to the element type on store.
 * Replaces swiglu_fwd<bf16,bf16,bf16> (swiglu.cu:397-525; kernel swiglu.cu:103-394). N is the FULL 2*ff as in
 * the reference; ldh is the row stride of H itself (the reference's operator passes ldC/2, swiglu.cu:414).
 */
FSW_API int fsw_gateup(int dtype, int64_t M, int64_t N, int64_t K,
               const void* X, int64_t ldx, const void* W13, int64_t ldw,
               void* H, int64_t ldh, void* stream);

/*
 * fsw_gateup whose H is float [M, N/2] (row stride ldh in floats, 4-byte aligned): the gated fp32 value is stored
 * as it is, with no rounding. Replaces swiglu_fwd<bf16,bf16,float>, the reference's build with C_TYPE float
 * (constants.cuh:9-14; cast_mmaresult's to_float branch, swiglu.cu:47-82; "C can work with either bf16 or fp32",
 * swiglu.cu:470-471). Inputs as for fsw_gateup.
 */
FSW_API int fsw_gateup_f32out(int dtype, int64_t M, int64_t N, int64_t K,
                      const void* X, int64_t ldx, const void* W13, int64_t ldw,
                      float* H, int64_t ldh, void* stream);

/* Host-only validation of fsw_down: M, D, FF >= 0; FF % 8 == 0; ldh >= FF, ldw2 >= FF, ldy >= D;
 * ldh % 8 == 0, ldw2 % 8 == 0; H, W2 16-byte aligned. */
FSW_API int fsw_validate_down(int dtype, int64_t M, int64_t D, int64_t FF,
                      const void* H, int64_t ldh, const void* W2, int64_t ldw2,
                      const void* Y, int64_t ldy);

/* Bytes of device scratch fsw_down needs for this shape: fp32 split-K partials where few output tiles meet a deep K
 * (FSW_E_WORKSPACE without them), 0 otherwise. Up to 256 rows less is accepted where K parts are only an option (few rows, a short K):
 * fsw_down and fsw_mlp then make as many parts as there is room for, which is slower. 4 * M * D bytes per part, at most 256 MB above 256 rows; the number of parts
 * follows the shape's fastest plan and may differ from one version to the next. No counterpart in the reference, which has no down projection. */
FSW_API size_t fsw_down_workspace_bytes(int dtype, int64_t M, int64_t D, int64_t FF);

/*
 * Y[M, D] = H[M, FF] @ W2[D, FF].T, fp32 accumulation, one RNE rounding on store.
 * No counterpart in the reference (its op ends at H, swiglu.cu:538-553); it is the `@ Wd` step of the
 * full MLP forward (silu(X@Wg) * (X@Wu)) @ Wd.
 */
FSW_API int fsw_down(int dtype, int64_t M, int64_t D, int64_t FF,
             const void* H, int64_t ldh, const void* W2, int64_t ldw2,
             void* Y, int64_t ldy,
             void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of device scratch fsw_mlp needs: the H[M, FF] intermediate (panel-blocked in the large-tile regime) plus the
 * scratch of its down projection. With 128 * M bytes more, rows of H are whole 128-byte lines where FF % 64 != 0 and M > 256: the
 * same result, 1 .. 6 % sooner (the torch module allocates that). */
FSW_API size_t fsw_mlp_workspace_bytes(int dtype, int64_t M, int64_t D, int64_t FF);

/*
 * Whole forward: Y[M, D] = (silu(X @ Wg) * (X @ Wu)) @ Wd as fsw_gateup followed by fsw_down on the same
 * stream, with H held in `workspace`. X is [M, D]; W13 is [2*FF, D]; W2 is [D, FF].
 */
FSW_API int fsw_mlp(int dtype, int64_t M, int64_t D, int64_t FF,
            const void* X, int64_t ldx, const void* W13, int64_t ldw13,
            const void* W2, int64_t ldw2, void* Y, int64_t ldy,
            void* workspace, size_t workspace_bytes, void* stream);

/*
 * fsw_mlp for callers that cannot allocate device memory at all (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc): same arguments without the workspace, same kernels, same result bit for
 * bit wherever fsw_mlp_workspace_bytes() is within the array (beyond, the down projection splits K less often, so that
 * its fp32 sums are taken in another order). No counterpart in the reference. The scratch (H, split-K partials and their ticket counters) lives in a static
 * device array of fsw_mlp_static_max_bytes() = 64 MiB inside the library, which every GPU the library runs on holds
 * until the process ends; shapes whose H alone exceeds it return FSW_E_STATIC_LIMIT (it covers
 * decode and small batches: at d = 4096, ff = 14336 every M <= 2340). The call itself allocates and frees nothing;
 * the first call on a device looks the array's address up (make it outside graph capture). All calls on one GPU share
 * the one array: calls that overlap in time on the same GPU (different streams, concurrent graph replays) race on
 * it and must be serialised by the caller. The single-launch decode option of fsw_set_variant is ignored here.
 */
FSW_API size_t fsw_mlp_static_max_bytes(void);
FSW_API int fsw_mlp_static(int dtype, int64_t M, int64_t D, int64_t FF,
                           const void* X, int64_t ldx, const void* W13, int64_t ldw13,
                           const void* W2, int64_t ldw2, void* Y, int64_t ldy, void* stream);

/* Text for an FSW_E_* code (static storage, never NULL). */
FSW_API const char* fsw_strerror(int code);

/*
 * Panel-blocked layout (no counterpart in the reference; it is the offline/in-flight layout transform that lets the
 * large-tile kernels fetch whole cache lines). A blocked copy of a row-major [rows, k] matrix is ceil(rows / 256)
 * panels of ceil(k / 32) blocks; block (panel, kt) is [256 rows][32 elements] contiguous (16 KB) and holds rows
 * 256 panel .. 256 panel + 255, columns 32 kt .. 32 kt + 31, zero padded. fsw_mlp uses it internally for M > 64 when
 * both projections run 256 x 256 tiles: H is written and read blocked (fsw_gateup_hblocked, fsw_down_blocked); X is
 * read row-major. The entry points below expose the steps, and let a caller block the weights ONCE (fsw_prepack_*)
 * and pass them with w_blocked = 1. Constraints as for fsw_gateup / fsw_down (K, FF and row-major leading dimensions multiples of 8,
 * 16-byte aligned bases); the blocked kernels are the 256 x 256 tiled kernels, whatever M is.
 */
FSW_API size_t fsw_blocked_bytes(int64_t rows, int64_t k);
FSW_API int fsw_block_rows(int dtype, int64_t rows, int64_t k, const void* src, int64_t ld, void* dst_blocked,
                           void* stream);
/* W13 [N, K] interleaved as in swiglu.cu:380-381 -> blocked, with each panel's 128 "up" rows first, then its 128
 * "gate" rows (the order the gated kernel keeps a weight tile in LDS). */
FSW_API int fsw_prepack_w13(int dtype, int64_t N, int64_t K, const void* W13, int64_t ldw, void* dst_blocked,
                            void* stream);
FSW_API int fsw_prepack_w2(int dtype, int64_t D, int64_t FF, const void* W2, int64_t ldw2, void* dst_blocked,
                           void* stream);
/* H[M, N/2] = gate/up of X_blocked[M, K]; W13 row-major (w_blocked = 0, ldw) or from fsw_prepack_w13 (1); H is
 * written blocked when ldh == 0 (for fsw_down_blocked), else row-major with row stride ldh. */
FSW_API int fsw_gateup_blocked(int dtype, int64_t M, int64_t N, int64_t K, const void* X_blocked, const void* W13,
                               int64_t ldw, int w_blocked, void* H, int64_t ldh, void* stream);
/* fsw_gateup on row-major X (row stride ldx) whose H is written blocked, for fsw_down_blocked: the two halves of
 * fsw_mlp in the large-tile regime. W13 row-major (w_blocked = 0, ldw) or from fsw_prepack_w13 (1). K > 0;
 * constraints as for fsw_gateup; H 16-byte aligned. */
FSW_API int fsw_gateup_hblocked(int dtype, int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx, const void* W13,
                                int64_t ldw, int w_blocked, void* H_blocked, void* stream);
/* Y[M, D] (row-major, ldy) = H_blocked[M, FF] @ W2^T; W2 row-major (0, ldw2) or from fsw_prepack_w2 (1). */
FSW_API int fsw_down_blocked(int dtype, int64_t M, int64_t D, int64_t FF, const void* H_blocked, const void* W2,
                             int64_t ldw2, int w_blocked, void* Y, int64_t ldy, void* stream);

/* fsw_gateup with a scratch argument, kept for callers written against it: the query returns 0 for every shape and
 * the call is fsw_gateup (the large-tile kernel reads row-major X in whole cache lines; no blocked copy is made). */
FSW_API size_t fsw_gateup_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K);
FSW_API int fsw_gateup_ws(int dtype, int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx, const void* W13,
                          int64_t ldw, void* H, int64_t ldh, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Attention beside the MLP (no counterpart in the reference, whose extension ends at the MLP): the other half of a decoder layer that is being
 * served. Hq query heads share Hkv key-value heads (Hq a multiple of Hkv, both at most 1024; query head h reads head
 * h / (Hq / Hkv)) of D channels (a multiple of 8, 8 .. 256). Rows of queries, keys, values and outputs are addressed by a token and a
 * head stride in elements, multiples of 8 and not negative, with D contiguous channels from a 16-byte aligned base: the slices of a fused
 * projection's output are such rows. Rows of an output must not overlap. At most 2^20 tokens per call.
 * Whole numbers on the device (positions, slots, pages, lengths, offsets) are int32. The host cannot check them, so the
 * kernels do: nothing outside the described arrays is ever read or written, and what each kernel does instead is said below.
 */

/* A paged cache of one layer. Token t of a page holds its head h at element page * page_stride + h * head_stride +
 * t * token_stride of k, and of v likewise. Strides are multiples of 8 below 2^40 (token_stride: at most 2^24); pages * page_size <= 2^30.
 * A cache that is written has cells that do not overlap, each dimension inside the next larger stride. */
typedef struct fsw_kv_cache {
  void* k;
  void* v;
  int64_t pages, page_size;
  int64_t page_stride, head_stride, token_stride;
} fsw_kv_cache;

/* Host-only validation of fsw_kv_append. 0 <= rot <= D, rot even. */
FSW_API int fsw_validate_kv_append(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot,
                                   const void* Q, int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head,
                                   const void* V, int64_t v_token, int64_t v_head, const float* cos_sin, int64_t table_rows,
                                   const int32_t* positions, const int32_t* slots, const void* Qout, int64_t qo_token,
                                   int64_t qo_head, const void* Kout, int64_t ko_token, int64_t ko_head,
                                   const fsw_kv_cache* cache);

/*
 * Rotates queries and keys by their positions and appends keys and values to the cache. The first `rot` channels are turned in pairs (a, b) =
 * (x[i], x[i + rot/2]), or (x[2i], x[2i+1]) if `interleaved`: a cos - b sin, b cos + a sin in fp32, one rounding. Row p of
 * cos_sin [table_rows, rot] holds position p's rot/2 cosines, then its sines (16-byte aligned; 4-byte where rot is no multiple of 8). Qout may be Q itself, Kout K itself or NULL.
 * Token t goes to slot slots[t] = page * page_size + place in the page; a slot outside the cache appends nothing (padding). Slots of one
 * call must differ. A position outside the table gives NaN in the turned channels.
 */
FSW_API int fsw_kv_append(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, int interleaved,
                          const void* Q, int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head,
                          const void* V, int64_t v_token, int64_t v_head, const float* cos_sin, int64_t table_rows,
                          const int32_t* positions, const int32_t* slots, void* Qout, int64_t qo_token, int64_t qo_head,
                          void* Kout, int64_t ko_token, int64_t ko_head, const fsw_kv_cache* cache, void* stream);

/* Host-only validation of fsw_attn_decode (all but the workspace). B <= 65535; scale a positive normal number, finite also times log2(e); table_ld >=
 * ceil(max_len / page_size), or 0: all sequences have the same pages. */
FSW_API int fsw_validate_attn_decode(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq,
                                     int64_t q_head, const fsw_kv_cache* cache, const int32_t* block_table, int64_t table_ld,
                                     const int32_t* lengths, int64_t max_len, float scale, const void* O, int64_t o_seq,
                                     int64_t o_head);

/* Bytes of device scratch fsw_attn_decode needs (FSW_E_WORKSPACE without them): the float32 sums of the parts that long sequences are
 * split into where there are few of them, else 0. Need not be initialised. */
FSW_API size_t fsw_attn_decode_workspace_bytes(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len);

/*
 * O[b, h] = softmax_j(scale * Q[b, h] . k_j) . v_j over the keys j < lengths[b] of sequence b, which lie in pages
 * block_table[b * table_ld + j / page_size]: one new token per sequence. fp32 scores and sums, weights in two elements
 * that hold 16 bits (bf16) or 22 (fp16) of them, one rounding. max_len: the host's bound of the lengths, which sets
 * the launch's shape. A length of 0 gives zeros; a length below 0 or above max_len, or a page outside the cache among a sequence's pages, gives NaN for that
 * sequence. What the cache holds behind a length is never used. Every key before it weighs more than nothing: an infinity among their values gives that
 * infinity, both signs or a NaN give NaN, in their channel. Finite values give finite sums, however large they are; in bf16 a weight
 * below 2^-88 of the largest may count as none or as that much, which values 2^80 times as large as the result would show.
 */
FSW_API int fsw_attn_decode(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                            const fsw_kv_cache* cache, const int32_t* block_table, int64_t table_ld, const int32_t* lengths,
                            int64_t max_len, float scale, void* O, int64_t o_seq, int64_t o_head, void* workspace,
                            size_t workspace_bytes, void* stream);

/* Host-only validation of fsw_attn_prompt. B <= 65535; k_token, v_token between D and 2^21; scale a positive normal number, finite also times log2(e). */
FSW_API int fsw_validate_attn_prompt(int dtype, int64_t Tq, int64_t Tk, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q,
                                     int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head,
                                     const void* V, int64_t v_token, int64_t v_head, const int32_t* cu_q, const int32_t* cu_k,
                                     float scale, const void* O, int64_t o_token, int64_t o_head);

/*
 * Causal attention of B packed sequences: sequence b is rows cu_q[b] .. cu_q[b + 1] - 1 of Q and O and rows cu_k[b] .. cu_k[b + 1] - 1 of
 * K and V (B + 1 offsets each, ascending from 0; for whole prompts both are one array). Ends are aligned: query i of nq sees the keys
 * j <= i + nk - nq. A query that sees no key, and a row of Q behind the last sequence, gives zeros. Scores, sums and the
 * normalisation are fp32; values of any size, infinities and NaN among them are as for fsw_attn_decode, and do not reach rows that do not see them;
 * the weights 2^(c s - m) are rounded to the element type once, for the matrix product with V, and their sum is taken of the rounded values.
 */
FSW_API int fsw_attn_prompt(int dtype, int64_t Tq, int64_t Tk, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q,
                            int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head, const void* V,
                            int64_t v_token, int64_t v_head, const int32_t* cu_q, const int32_t* cu_k, float scale, void* O,
                            int64_t o_token, int64_t o_head, void* stream);

/* Rows, (token, query head of a key-value head) pairs, of a workgroup of fsw_attn_prompt: 64 where the launch is small, else 128; 0 for what it refuses or where
 * there is nothing to launch. For tests and benchmarks. */
FSW_API int fsw_attn_prompt_rows(int dtype, int64_t Tq, int64_t B, int64_t Hq, int64_t Hkv, int64_t D);

/*
 * The same cache in 8 bits. A row (one token, one head, keys or values) is D e4m3 elements c_i (four significant bits, 2^-9 .. 448, no
 * infinities) and one power of two: it stands for c_i 2^e. Elements are addressed as in fsw_kv_cache (strides in elements, multiples of 16; D a
 * multiple of 16); the scale of token t of a page's head h is byte page * scale_page_stride + h * scale_head_stride + t *
 * scale_token_stride of k_scale (v_scale), e + 127 (e8m0; 255 is no number). Scales that 16 tokens have side by side, in aligned words, are read faster.
 */
typedef struct fsw_kv_cache8 {
  void* k;
  void* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t pages, page_size;
  int64_t page_stride, head_stride, token_stride;
  int64_t scale_page_stride, scale_head_stride, scale_token_stride;
} fsw_kv_cache8;

/* Host-only validation of fsw_kv_append8: as for fsw_kv_append. */
FSW_API int fsw_validate_kv_append8(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot,
                                    const void* Q, int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head,
                                    const void* V, int64_t v_token, int64_t v_head, const float* cos_sin, int64_t table_rows,
                                    const int32_t* positions, const int32_t* slots, const void* Qout, int64_t qo_token,
                                    int64_t qo_head, const void* Kout, int64_t ko_token, int64_t ko_head, const void* Vout,
                                    int64_t vo_token, int64_t vo_head, const fsw_kv_cache8* cache);

/*
 * fsw_kv_append to a cache in 8 bits: e is the least integer, -126 at least, with max |x_i| <= 448 2^e over the row's finite values (0 for a row of
 * zeros), c_i = x_i 2^-e rounded to nearest, ties to even. Infinities and NaN become NaN; a value that would round above the element type's
 * largest becomes the largest below. Keys are rotated in 64 bits and rounded once. Kout and Vout (each may be NULL) receive the
 * rows as the cache holds them, in the element type: what a prompt should attend to, so that it sees what later tokens will. Qout may be Q itself, Kout K itself, Vout V
 * itself.
 */
FSW_API int fsw_kv_append8(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, int interleaved,
                           const void* Q, int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head,
                           const void* V, int64_t v_token, int64_t v_head, const float* cos_sin, int64_t table_rows,
                           const int32_t* positions, const int32_t* slots, void* Qout, int64_t qo_token, int64_t qo_head,
                           void* Kout, int64_t ko_token, int64_t ko_head, void* Vout, int64_t vo_token, int64_t vo_head,
                           const fsw_kv_cache8* cache, void* stream);

/* Host-only validation of fsw_kv_read and fsw_kv_read8. B <= 65535; width >= 0, table_ld >= width, or 0. */
FSW_API int fsw_validate_kv_read(int dtype, int64_t T, int64_t B, int64_t Hkv, int64_t D, const fsw_kv_cache* cache, const int32_t* block_table,
                                 int64_t table_ld, int64_t width, const int32_t* cu, const void* Kout, int64_t ko_token, int64_t ko_head,
                                 const void* Vout, int64_t vo_token, int64_t vo_head);
FSW_API int fsw_validate_kv_read8(int dtype, int64_t T, int64_t B, int64_t Hkv, int64_t D, const fsw_kv_cache8* cache, const int32_t* block_table,
                                  int64_t table_ld, int64_t width, const int32_t* cu, const void* Kout, int64_t ko_token, int64_t ko_head,
                                  const void* Vout, int64_t vo_token, int64_t vo_head);

/*
 * Keys and values of B sequences out of their pages, packed: row cu[b] + j of Kout and Vout (cu[b] <= row < cu[b + 1]; B + 1 offsets, ascending from
 * 0) is token j of sequence b, which lies in page block_table[b * table_ld + j / page_size], j / page_size < width. For fsw_attn_prompt, whose prompts may continue
 * what is in the cache. Rows behind the last sequence are zeros; a token behind the table's row, or in a page outside the cache, is NaN. Of a cache in 8 bits:
 * c_i 2^e rounded to the element type.
 */
FSW_API int fsw_kv_read(int dtype, int64_t T, int64_t B, int64_t Hkv, int64_t D, const fsw_kv_cache* cache, const int32_t* block_table,
                        int64_t table_ld, int64_t width, const int32_t* cu, void* Kout, int64_t ko_token, int64_t ko_head, void* Vout,
                        int64_t vo_token, int64_t vo_head, void* stream);
FSW_API int fsw_kv_read8(int dtype, int64_t T, int64_t B, int64_t Hkv, int64_t D, const fsw_kv_cache8* cache, const int32_t* block_table,
                         int64_t table_ld, int64_t width, const int32_t* cu, void* Kout, int64_t ko_token, int64_t ko_head, void* Vout,
                         int64_t vo_token, int64_t vo_head, void* stream);

/* fsw_attn_decode over a cache in 8 bits: the same checks, scratch rules and answers to invalid sequences. A row whose scale is 255 is NaN. Keys are
 * taken rounded to the queries' type. Values below 2^-100 lose bits (their weights times their scales are held in numbers from 2^-133 on). */
FSW_API int fsw_validate_attn_decode8(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq,
                                      int64_t q_head, const fsw_kv_cache8* cache, const int32_t* block_table, int64_t table_ld,
                                      const int32_t* lengths, int64_t max_len, float scale, const void* O, int64_t o_seq,
                                      int64_t o_head);
FSW_API size_t fsw_attn_decode8_workspace_bytes(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len);
FSW_API int fsw_attn_decode8(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                             const fsw_kv_cache8* cache, const int32_t* block_table, int64_t table_ld, const int32_t* lengths,
                             int64_t max_len, float scale, void* O, int64_t o_seq, int64_t o_head, void* workspace,
                             size_t workspace_bytes, void* stream);

/* Host-only validation of fsw_attn_shared and fsw_attn_shared8 (all but the workspace): as for fsw_attn_decode; prefix_len >= 0, prefix_len + max_len <= 2^30. */
FSW_API int fsw_validate_attn_shared(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq,
                                     int64_t q_head, const fsw_kv_cache* cache, const int32_t* prefix, int64_t prefix_len,
                                     const int32_t* block_table, int64_t table_ld, const int32_t* lengths, int64_t max_len,
                                     float scale, const void* O, int64_t o_seq, int64_t o_head);
FSW_API int fsw_validate_attn_shared8(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq,
                                      int64_t q_head, const fsw_kv_cache8* cache, const int32_t* prefix, int64_t prefix_len,
                                      const int32_t* block_table, int64_t table_ld, const int32_t* lengths, int64_t max_len,
                                      float scale, const void* O, int64_t o_seq, int64_t o_head);

/* Bytes of device scratch fsw_attn_shared (fsw_attn_shared8) needs (FSW_E_WORKSPACE without them): float32 sums of the shares of the prefix and of
 * the sequences' own keys. Need not be initialised. */
FSW_API size_t fsw_attn_shared_workspace_bytes(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t max_len);
FSW_API size_t fsw_attn_shared8_workspace_bytes(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t max_len);

/*
 * fsw_attn_decode for a batch whose sequences all begin with the same prefix_len tokens, which are read once for all of them: they lie in pages
 * prefix[j / page_size], j < prefix_len. lengths, max_len and block_table are of each sequence's own tokens, which begin with a page of their own
 * and follow the prefix. A length of 0 leaves the prefix alone. The weights of the prefix are rounded to the element type once, for the matrix product, and their
 * sum is taken of the rounded values, as in fsw_attn_prompt; infinities, NaN, lengths and pages of own tokens are as for fsw_attn_decode; a
 * page outside the cache among the prefix's gives NaN for all. fsw_attn_shared8 takes the prefix's keys and values rounded to the element type.
 */
FSW_API int fsw_attn_shared(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                            const fsw_kv_cache* cache, const int32_t* prefix, int64_t prefix_len, const int32_t* block_table,
                            int64_t table_ld, const int32_t* lengths, int64_t max_len, float scale, void* O, int64_t o_seq,
                            int64_t o_head, void* workspace, size_t workspace_bytes, void* stream);
FSW_API int fsw_attn_shared8(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                             const fsw_kv_cache8* cache, const int32_t* prefix, int64_t prefix_len, const int32_t* block_table,
                             int64_t table_ld, const int32_t* lengths, int64_t max_len, float scale, void* O, int64_t o_seq,
                             int64_t o_head, void* workspace, size_t workspace_bytes, void* stream);

/* Rows, (sequence, query head of a key-value head) pairs, of a workgroup over the prefix of fsw_attn_shared (fsw_attn_shared8): 64, 128 or 256 by the plan of
 * least estimated time, but 64 where the page size is no multiple of the keys that a wave loads at a time; 0 for what is refused or where there is no prefix. For
 * tests and benchmarks. */
FSW_API int fsw_attn_shared_rows(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t page_size);
FSW_API int fsw_attn_shared8_rows(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t page_size);

/* Host-only validation of fsw_add_norm. M <= 2^30; D a multiple of 8 up to 32768; leading dimensions multiples of 8, those of results at least D, pointers
 * 16-byte aligned; scale finite, eps a positive normal number. */
FSW_API int fsw_validate_add_norm(int dtype, int64_t M, int64_t D, const void* X, int64_t ldx, const void* Y, int64_t ldy, const void* gate,
                                  int64_t ld_gate, const void* post, const void* pre, float scale, float eps, const void* Xout,
                                  int64_t ldxo, const void* H, int64_t ldh);

/*
 * The norms around a block of a layer, its gate and its residual scale, a row at a time:
 *   b = Y rms(Y) post,  Xout = X + scale gate b,  H = Xout rms(Xout) pre,  rms(z) = (mean z^2 + eps)^(-1/2)
 * in fp32 (squares in 64 bits), Xout and H rounded once each, H from the unrounded Xout. post, pre: D weights. post NULL: b = Y. pre NULL: weights of 1. gate: a row for
 * every row (ld_gate >= D) or one for all (ld_gate = 0); NULL: 1. Y NULL (then gate and post are, too): H alone of X, for the norm before the first block. One of Xout and H may
 * be NULL. Xout may be X itself, H may be Y itself, with the same leading dimension.
 */
FSW_API int fsw_add_norm(int dtype, int64_t M, int64_t D, const void* X, int64_t ldx, const void* Y, int64_t ldy, const void* gate,
                         int64_t ld_gate, const void* post, const void* pre, float scale, float eps, void* Xout, int64_t ldxo,
                         void* H, int64_t ldh, void* stream);

/* The hipError_t (as int) of the most recent failed launch on the calling thread, 0 if none. */
FSW_API int fsw_last_hip_error(void);

/* ABI version: major * 1000 + minor. 2000: the measurement kernels fsw_probe_* left this library (libfsw_probe.so,
 * fsw_probe.h); fsw_gateup_f32out and fsw_gateup_hblocked joined it; fsw_gateup_workspace_bytes returns 0. 2001: the attention
 * entry points. 2002: fsw_attn_prompt_rows. 2003: the cache in 8 bits, fsw_kv_read, fsw_attn_shared, fsw_add_norm. 2004:
 * fsw_attn_shared_rows, fsw_attn_shared8_rows. */
FSW_API int fsw_version(void);

/*
 * Kernel-selection override for tests and tuning, PER CALLING THREAD (thread-local): it changes the kernel choice
 * of later calls made by the same thread only, so a thread's fsw_*_workspace_bytes() queries and the launches
 * that follow them always agree. family: 0 = gate/up, 1 = down; variant < 0 restores the automatic choice by
 * shape; 0 .. 5 force one tiled kernel (dma_128x128, dma8w_128x256, dma_128x192, dma8w_128x256 again, dma_128x64,
 * pair16_256x256; a forced kernel runs unsplit and needs no scratch); 100 is the weight-streaming kernel (honoured
 * for M <= 64; the dispatcher itself picks it up to 16 .. 48 rows, the larger the weights the fewer); 102 is the
 * persistent streaming kernel (honoured for M <= 16; automatic only for d * ff >= 2^27); family 0 variant 101
 * makes fsw_mlp run M <= 16 as ONE persistent launch (gate/up, device-wide barrier, down) instead of two launches
 * -- see fsw_decode_barrier_failures(): a correctness-tested experiment that measures SLOWER than the two launches
 * (69.7 vs 61.0 us at M = 16, d = 4096, ff = 14336) and is kept for study only; 103 is 101 with a barrier that cannot
 * complete, a hook of the failure-path test that is refused (FSW_E_VARIANT) unless the environment holds
 * FSW_TEST_HOOKS=1;
 * variants 115, 116, 117 = the 256-row kernel with 160, 192, 224 activation rows per tile (row-major operands);
 * family 1 variant 104 makes fsw_mlp run the down projection of M <= 32 rows on the split-K streaming kernel
 * (32-row tiles, two K ranges whose partial tiles meet through ticket counters that the gate/up kernel zeroes)
 * whatever the shape (nothing selects it by itself: K parts on the producer / consumer kernel are faster);
 * variants 200 + i = tile i of the producer / consumer kernel, whole tiles.
 * Returns FSW_E_VARIANT for unknown ids.
 */
FSW_API int fsw_set_variant(int family, int variant);

/*
 * The single-launch decode forward (fsw_set_variant(0, 101)) synchronises its workgroups with a device-wide barrier,
 * which completes only if all of them are resident at once. The wait is bounded: when other work holds compute units
 * the kernel gives up, skips the down projection (Y is left incomplete, never computed from a partial H) and marks
 * its barrier slot. This call returns how many such launches there were on the current device since it was last
 * called and clears the marks, or a negative FSW_E_* code. It copies synchronously: call it after synchronising the
 * stream, with no single-launch forward in flight. A caller that opts into variant 101 must check it before using Y.
 * With 64 single-launch forwards in flight, or on a stream that is being captured into a graph, fsw_mlp runs the
 * two-launch path instead. No counterpart in the reference.
 */
FSW_API int fsw_decode_barrier_failures(void);

/* Families 0 (gate/up), 1 (fsw_down) and 2 (the down projection inside fsw_mlp): name of the dispatcher's range that this
 * shape falls in (static storage): "skinny", "decode_stream" (up to 48 rows, weight streaming), "stream_split" (17 .. 32 rows of
 * large layers inside fsw_mlp), "dma_*" (up to 64, 128, 192, 256 rows to share the weights, and small problems), "pair16_*"
 * (tiles of 256 weight rows); "splitk_<name>" when the down projection splits K. What fsw_set_variant forces has these names.
 * Families 3, 4 and 5 (of 0, 1 and 2): the kernel that runs there, for operands whose rows are as long as K_or_FF: "mid_<rows of
 * weights>x<rows of activations>" for the producer / consumer kernel, which serves most of the first four ranges, else the name
 * above. */
FSW_API const char* fsw_variant_name(int family, int dtype, int64_t M, int64_t N_or_D, int64_t K_or_FF);

#ifdef __cplusplus
}
#endif
#endif /* FSW_H */
