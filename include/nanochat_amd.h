/*
 * nanochat_amd: the C ABI of the MI355X (gfx950) fp8 KV-cache decode path.
 *
 * Every pointer argument is a device address unless stated otherwise; sizes are element counts. Every
 * entry point is stream-ordered on `stream` (a hipStream_t; NULL = the null stream) and never
 * synchronizes. Entry points that return int return NC_OK (0), a negative NC_ERR_* code for an argument
 * the host can check, or a positive hipError_t from the launch.
 *
 * Data formats (the build's; the reference caches bf16, model/kernels/decode.cu:726):
 *   bf16             raw 16-bit patterns (torch.bfloat16 storage)
 *   k_pages, v_pages uint8 [num_pages][Hkv][2048]: one 16-token page of one KV head, OCP e4m3fn codes in
 *                    the MFMA tiling documented in nanochat_amd/csrc/nc_device.h (k/v_page_offset)
 *   kv_scale         fp32 [num_pages][Hkv][2][16]: one absmax/448 scale per (token, KV head), K scales then
 *                    V scales of a page's 16 slots (one 128-byte line per page and head)
 *   block_table      int32 [B][max_pages]: position p of sequence b is slot p % 16 of page
 *                    block_table[b][p / 16]
 * Query head h reads KV head h / (Hq / Hkv); Hq must be a multiple of Hkv with Hq / Hkv <= 16.
 */
#ifndef NANOCHAT_AMD_H
#define NANOCHAT_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    NC_OK = 0,
    NC_ERR_NULL = -1,       /* a required pointer is NULL */
    NC_ERR_SHAPE = -2,      /* a size or head count out of the supported range */
    NC_ERR_WORKSPACE = -3,  /* the workspace is smaller than its nc_*_workspace_bytes, or not aligned as asked */
};

/* Text of a status code (static storage). */
const char *nc_status_string(int status);

/* Version of this ABI (bumped on any signature or format change). */
int nc_abi_version(void);

/*
 * Training-form fused q/k prologue; same symbol, arguments and meaning as the reference's
 * model/kernels/qk_prologue.cu:111-118 (called by model/ops/qk_prologue.py:13-21 qk_forward):
 * q, k: bf16 (B, T, H, 128) views with token stride 3*H*128 (the fused projection); gq, gk: fp32 [128];
 * qo, ko: bf16 contiguous (B, T, H, 128); cos, sin: fp32 [T][64] indexed by the token's position t;
 * rows = B*T*H. Per row: RMS norm (eps FLT_EPSILON), gain, -theta rotation, one bf16 rounding.
 * Like the reference it returns nothing; nc_last_error() reports its launch status.
 */
void qkp_forward(const void *q, const void *k, const void *gq, const void *gk, void *qo, void *ko, const void *cos,
                 const void *sin, long long rows, int H, int T, void *stream);

/* The prologue's backward: the reference's qkp_backward (model/kernels/qk_prologue.cu:128-136), same arguments.
 * q, k as for qkp_forward; dqo, dko: the outputs' gradients, contiguous [rows][128] bf16; dq, dk: the inputs'
 * gradients at q's and k's strides (token stride 3 H 128); dgq, dgk: the gains' gradients fp32 [128], summed in a
 * fixed order (bitwise reproducible); part: fp32 [2 qkp_backward_blocks()][128] scratch. rows = 0 is allowed (the
 * gain gradients are zero). Returns nothing; nc_last_error() reports the status. */
void qkp_backward(const void *q, const void *k, const void *gq, const void *gk, const void *dqo, const void *dko,
                  void *dq, void *dk, void *dgq, void *dgk, void *part, const void *cos, const void *sin,
                  long long rows, int H, int T, void *stream);

/* Blocks per tensor of qkp_backward's partial gain gradients (reference qk_prologue.cu:120-125): fixed. */
int qkp_backward_blocks(void);

/*
 * Value-embedding gate and mix of training; same symbols, arguments and meaning as the reference's
 * model/kernels/ve_gate.cu:199-214 (called by model/ops/ve_gate.py:13-33), with the reference's fixed shape H = 6
 * heads, C = 768. Forward: n bf16 [rows][C] (the normed stream), v bf16 rows at v_stride elements, idx int32 [rows],
 * table fp32 [vocab][C], w fp32 [H][C] -> out bf16 [rows][C] = v + gate[head] * bf16(table[idx]),
 * gate fp32 [rows][H] = 2 sigmoid(n w^T). Backward: dout bf16 rows at dout_stride, ids int32 [rows] sorted tokens
 * (equal tokens must be adjacent, else the table gradient is undefined), order int64 [rows] their rows (a row
 * outside [0, rows) is skipped), gate from the forward -> dn bf16 [rows][C], dz bf16 [rows][H] (dw = dz^T n is the
 * caller's GEMM), and the table's gradient added into dtable fp32 [vocab][C]. Tokens are trusted (negative ones
 * read as a zero embedding). Like the reference they return nothing; nc_last_error() reports the status.
 */
void ve_forward(const void *n, const void *v, long long v_stride, const void *idx, const void *table, const void *w,
                void *out, void *gate, long long rows, void *stream);
void ve_backward(const void *dout, long long dout_stride, const void *ids, const void *order, const void *table,
                 const void *w, const void *gate, void *dn, void *dtable, void *dz, long long rows, void *stream);

/* ve_forward / ve_backward for any head count 1 <= heads <= 16 (C = 128 heads) and a table of `vocab` rows: a token
 * outside [0, vocab) mixes in nothing and receives no gradient. Strides are multiples of 8 elements and at least C;
 * n, v, table, w, out, dout, dn and dtable are 16-byte aligned. rows = 0 launches nothing. */
int nc_ve_forward(const void *n, const void *v, long long v_stride, const int32_t *idx, const float *table,
                  long long vocab, const float *w, void *out, float *gate, long long rows, int heads, void *stream);
int nc_ve_backward(const void *dout, long long dout_stride, const int32_t *ids, const int64_t *order,
                   const float *table, long long vocab, const float *w, const float *gate, void *dn, float *dtable,
                   void *dz, long long rows, int heads, void *stream);

/* The gate weight's gradient dw [heads][C] = dz^T n in fp32, summed in a fixed order: dz bf16 [rows][heads] (of
 * nc_ve_backward), n bf16 [rows][C] contiguous, 8-byte aligned; rows >= 1. workspace:
 * nc_ve_weight_grad_workspace_bytes (0 for no rows, -1 for sizes it does not take). */
long long nc_ve_weight_grad_workspace_bytes(long long rows, int heads);
int nc_ve_weight_grad(const void *dz, const void *n, long long rows, int heads, float *dw, void *workspace,
                      long long workspace_bytes, void *stream);

/*
 * Training attention forward: the varlen causal attention the reference runs through FlashAttention-4
 * (model/ops/flash_attn.py:340-345, _flash_attn_fwd(q, k, v, cu_seqlens, cu_seqlens, T, T, causal=True,
 * window_size_left=window, return_lse=True)). q, k, v: bf16 (total, heads, 128) with contiguous heads at token strides
 * q_stride, k_stride, v_stride (elements, multiples of 8); cu_seqlens: int32 [segments + 1] (segment s is tokens
 * cu[s] .. cu[s+1] - 1, at most max_seqlen of them). Row i of a segment attends keys j of the same segment with
 * j <= i and i - j <= window (window < 0: no left limit), scores scaled by softmax_scale.
 * out: bf16 (total, heads, 128) contiguous; lse: fp32 [heads][lse_stride], ln of the row's sum of exponentials.
 */
int nc_flash_attn_fwd(const void *q, const void *k, const void *v, long long q_stride, long long k_stride,
                      long long v_stride, const int32_t *cu_seqlens, int segments, int max_seqlen, int heads,
                      int window, float softmax_scale, void *out, float *lse, long long lse_stride, void *stream);

/*
 * Training attention backward (the reference's _flash_attn_bwd and bwd_bf16dq, model/ops/flash_attn.py:367-391):
 * q, k, v, dout as the forward's inputs and the output's gradient (token strides in elements); lse from
 * nc_flash_attn_fwd; dpsum fp32 (total, heads): D = dout . out per row (the reference's `rows`; see
 * nc_flash_attn_bwd_rows). Writes dq, dk, dv: bf16 (total, heads, 128) with contiguous heads at their token strides.
 * No atomics: the result does not depend on scheduling.
 */
int nc_flash_attn_bwd(const void *q, const void *k, const void *v, const void *dout, long long q_stride,
                      long long k_stride, long long v_stride, long long do_stride, const float *lse, long long lse_stride,
                      const float *dpsum, const int32_t *cu_seqlens, int segments, int max_seqlen, int heads,
                      int window, float softmax_scale, void *dq, void *dk, void *dv, long long dq_stride,
                      long long dk_stride, long long dv_stride, void *stream);

/* dpsum (total, heads) fp32 = sum over the 128 dims of dout * out (token strides in elements, even). */
int nc_flash_attn_bwd_rows(const void *out, long long o_stride, const void *dout, long long do_stride,
                           long long total, int heads, float *dpsum, void *stream);

/*
 * The training block's output projection with its residual and row statistic (the reference's residual_rms,
 * model/ops/linear.py:93-100): s = x w^T + res in fp32, out = bf16(s), rstd = 1 / sqrt(mean(s^2) + FLT_EPSILON). x bf16
 * [rows][k], w bf16 [n][k], res and out bf16 [rows][n], rstd fp32 [rows]; k a multiple of 128, n of 4; x and w 16-byte,
 * res and out 8-byte aligned. workspace: fp32 [rows][ceil(n / 32)].
 */
int nc_linear_residual_rms(const void *x, const void *w, const void *res, long long rows, int n, int k, void *out,
                           float *rstd, void *workspace, long long workspace_bytes, void *stream);

/* out[i][j] += sum over rows of a[row][i] b[row][j]: a bf16 [rows][n1], b bf16 [rows][n2], out fp32 [n1][n2] (n1, n2
 * multiples of 8; everything 16-byte aligned), summed in a fixed order. workspace: nc_weight_grad_workspace_bytes (-1
 * for sizes it does not take), 16-byte aligned. */
long long nc_weight_grad_workspace_bytes(long long rows, int n1, int n2);
int nc_weight_grad(const void *a, const void *b, long long rows, int n1, int n2, float *out, void *workspace,
                   long long workspace_bytes, void *stream);

/* Status of the last void entry point's launch on this host thread (NC_OK or a hipError_t). */
int nc_last_error(void);

/*
 * Quantize and append T new tokens per sequence to the paged fp8 cache. Replaces the cache store of the
 * reference's k_prologue (model/kernels/decode.cu:551-565, `kc/vc[cs][p] = bf16(k/v)`).
 * k, v: bf16 [B][T][Hkv][128] at token stride `token_stride` elements (batch stride T*token_stride);
 * token t of sequence b is written at position start_pos[b] + t; num_new (nullable) limits sequence b to
 * its first num_new[b] tokens. Per (token, KV head): scale = max|x| / 448 (1 if all zero),
 * code = e4m3fn_rne(clamp(x / scale, +-448)). Tokens whose page lies outside the block table or the
 * page pool are skipped.
 */
int nc_kv_append_fp8(const void *k, const void *v, long long token_stride, int B, int T, int Hkv,
                     const int32_t *start_pos, const int32_t *num_new, const int32_t *block_table, int max_pages,
                     void *k_pages, void *v_pages, float *kv_scale, int num_pages, void *stream);

/*
 * The fused append of a decode or prefill step: the reference's attn_prologue q/k math
 * (model/kernels/decode.cu:478-507 via qk_row.cuh:26-51) followed by nc_kv_append_fp8's quantized store.
 * qkv: bf16 [B][T][(Hq + 2*Hkv)*128] at token stride `token_stride` elements: q heads, then k heads, then
 * v heads. q and k rows are RMS-normed (eps FLT_EPSILON), multiplied by q_gain / k_gain (fp32 [128]) and
 * rotated by -theta with cos, sin (fp32 [rope_len][64]) at the token's position, then rounded to bf16;
 * q goes to q_out (bf16 [B][T][Hq][128], contiguous), k and v (unchanged) are quantized into the cache.
 * Tokens at positions >= rope_len are skipped.
 */
int nc_qk_norm_rope_append_fp8(const void *qkv, long long token_stride, int B, int T, int Hq, int Hkv,
                               const int32_t *start_pos, const int32_t *num_new, const float *q_gain,
                               const float *k_gain, const float *cos, const float *sin, int rope_len, void *q_out,
                               const int32_t *block_table, int max_pages, void *k_pages, void *v_pages,
                               float *kv_scale, int num_pages, void *stream);

/*
 * nc_qk_norm_rope_append_fp8 for packed rows, any number a sequence: row n of qkv (bf16 [rows][(Hq + 2 Hkv) 128] at
 * token_stride elements) is the token at position positions[n] and its K and V go to cache slot slot_map[n] = 16 page +
 * position % 16 (int32 [rows]; nc_pages_extend makes both), with the same bits; q goes to q_out (bf16 [rows][Hq][128]). A
 * row whose slot lies outside [0, 16 num_pages) or whose position lies outside [0, rope_len) is skipped: its q_out row
 * stays as it was. The slots of one call must differ. rows < 2^28, num_pages <= (2^31 - 1) / 16; no rows launch nothing.
 */
int nc_qk_norm_rope_append_rows_fp8(const void *qkv, long long token_stride, long long rows, int Hq, int Hkv,
                                    const int32_t *positions, const int32_t *slot_map, const float *q_gain,
                                    const float *k_gain, const float *cos, const float *sin, int rope_len, void *q_out,
                                    void *k_pages, void *v_pages, float *kv_scale, int num_pages, void *stream);

/* Workspace bytes nc_decode_attn_fp8 and nc_decode_step_fp8 need for these sizes (0 for unsupported sizes): fp32
 * partial results from its start and, in its last 1/256, one int32 arrival count per (sequence, KV head). The
 * workspace must be zero-filled before its first call and passed with the same workspace_bytes to every call: the
 * counts' place depends on that size alone, partials never go there and every call returns the counts it used to
 * zero, so one zero fill serves any number of calls of any sizes that fit, ordered on one stream. */
size_t nc_decode_workspace_bytes(int B, int Hq, int Hkv, int max_seq_len, int window);

/*
 * Single-token decode attention over the paged fp8 cache. Replaces the reference's k_attn
 * (model/kernels/decode.cu:567-675): sequence b's query at position p = seq_lens[b] - 1 attends keys
 * [max(p - window, 0), p] (window < 0: all), scores (q . k) * sm_scale, fp32 softmax, out bf16.
 * The current token must already be appended (nc_kv_append_fp8 / nc_qk_norm_rope_append_fp8).
 * q: bf16 [B][Hq][128]; out: bf16 [B][Hq][128]; seq_lens: int32 [B] (<= 0: inactive, output zeros; more
 * than max_seq_len: output NaN); max_seq_len <= max_pages * 16; B <= 4096.
 * Work split: a (sequence, KV head)'s keys are cut at every multiple of 1,024 positions, or of 256 positions when its
 * keys span at most 67 pages (1,072 positions); a last piece under 64 positions joins the one before it. Each piece
 * is one work item with its own softmax state; the wave that finishes a unit's last piece merges its pieces in
 * position order, in the same launch (one kernel). The split points depend on nothing but the sequence's own length, so its
 * output bits do not depend on the other sequences of the launch, on its place in the batch or on `workers` (waves
 * taking the items; 0: every wave slot of the device). The workspace (at least nc_decode_workspace_bytes) must be
 * zero-filled before its first use and keep one workspace_bytes value across calls.
 * A block-table entry outside [0, num_pages) makes that sequence's output NaN instead of reading outside
 * the pool.
 */
int nc_decode_attn_fp8(const void *q, const void *k_pages, const void *v_pages, const float *kv_scale,
                       const int32_t *block_table, int max_pages, int num_pages,
                       const int32_t *seq_lens, int max_seq_len, int B, int Hq, int Hkv, int window, float sm_scale,
                       int workers, void *out, void *workspace, size_t workspace_bytes, void *stream);

/*
 * The fused decode step: nc_qk_norm_rope_append_fp8 with T = 1 followed by nc_decode_attn_fp8, in one launch, with
 * the same results bit for bit (query rows, cache bytes and scales, attention output). Replaces the reference's
 * k_prologue + k_attn pair of a decode step (model/kernels/decode.cu:551-675, launched at 861-863). Sequence b's
 * token sits at position p = seq_lens[b] - 1 (seq_lens <= 0: inactive, nothing appended, output zeros); its row of
 * qkv (bf16 [B][(Hq + 2 Hkv) 128] at token_stride elements) is normed, rotated (q_gain, k_gain, cos, sin as in
 * nc_qk_norm_rope_append_fp8; rope_len >= max_seq_len) and, when ve is not NULL, its value row gets the value
 * embedding of token ve_tokens[b] (ve bf16 [ve_rows][C], ve_gate fp32 [Hkv][C], ve_h bf16 [B][C] the layer's normed
 * input; v += 2 sigmoid(ve_gate[kvh] . h) ve[token][kvh 128 ..]; a token outside [0, ve_rows) mixes nothing); k and v are quantized into the cache and q goes to
 * q_out (bf16 [B][Hq][128]) unless q_out is NULL; then the query attends as in nc_decode_attn_fp8. A sequence longer
 * than max_seq_len gets NaN and no append. The page receiving a sequence's token must not appear in another
 * sequence's block-table row (the work item that streams that page takes the token from registers while it stores
 * it). Workspace as for nc_decode_attn_fp8.
 */
int nc_decode_step_fp8(const void *qkv, long long token_stride, int B, int Hq, int Hkv, const int32_t *seq_lens,
                       const float *q_gain, const float *k_gain, const float *cos, const float *sin, int rope_len,
                       void *q_out, const void *ve_h, const void *ve, const float *ve_gate, const int32_t *ve_tokens,
                       int C, int ve_rows, const int32_t *block_table, int max_pages, void *k_pages, void *v_pages, float *kv_scale,
                       int num_pages, int max_seq_len, int window, float sm_scale, int workers, void *out,
                       void *workspace, size_t workspace_bytes, void *stream);

/* Bytes of the static device workspace of nc_decode_attn_fp8_noalloc (one array per GPU, held until the process
 * ends). */
#define NC_DECODE_SCRATCH_BYTES (16u << 20)

/*
 * No counterpart in the reference. For callers that cannot allocate device memory (code under HIP graph capture,
 * tight serving loops, harnesses that forbid hipMalloc): nc_decode_attn_fp8 with the same arguments, results and
 * errors, but its workspace is a static device array of NC_DECODE_SCRATCH_BYTES per GPU instead of the caller's. It
 * calls no allocating routine. A launch that needs more than that (nc_decode_workspace_bytes) returns
 * NC_ERR_WORKSPACE. Every call on one GPU shares that GPU's array: calls that overlap on one GPU (two streams, two
 * host threads) race and give undefined results; calls ordered on one stream do not.
 */
int nc_decode_attn_fp8_noalloc(const void *q, const void *k_pages, const void *v_pages, const float *kv_scale,
                               const int32_t *block_table, int max_pages, int num_pages, const int32_t *seq_lens,
                               int max_seq_len, int B, int Hq, int Hkv, int window, float sm_scale, int workers,
                               void *out, void *stream);

/*
 * Chunked-prefill attention over the paged fp8 cache (MFMA). Replaces the reference's prefill rows
 * (model/kernels/decode.cu:1041-1051 with enqueue_body's append-then-attend order, 859-863): row t of
 * sequence b sits at position start_pos[b] + t and attends keys [max(p - window, 0), p]; the chunk must
 * already be appended. q, out: bf16 [B][T][Hq][128].
 */
int nc_prefill_attn_fp8(const void *q, const void *k_pages, const void *v_pages, const float *kv_scale,
                        const int32_t *block_table, int max_pages, int num_pages,
                        const int32_t *start_pos, int B, int T, int Hq, int Hkv, int window, float sm_scale,
                        void *out, void *stream);

/* Workspace bytes nc_packed_attn_fp8 needs for these sizes, whatever the lengths on the device (0 for unsupported sizes):
 * partial results, and counts in its last 1/256. 16-byte aligned, else (as where it is too small) NC_ERR_WORKSPACE. As
 * nc_decode_workspace_bytes's: zero-filled before its first call and passed with the same workspace_bytes to every call, by
 * calls ordered on one stream; one workspace may serve both. Since the lengths are not known it holds the most partials
 * there can be, 32 or 128 query columns of 520 bytes each for every chunk of keys: 44 MB for 64 sequences of one row, 16 / 4
 * heads and 8,192 keys at most, but 1.4 GB for 256 of one row, 32 / 8 heads and 32,768 keys, and 5.5 GB with 8,192 rows.
 * A smaller max_seq_len (or a window) makes it smaller; up to 2,048 keys no partials are kept. */
size_t nc_packed_workspace_bytes(long long rows, int B, int Hq, int Hkv, int max_seq_len, int window);

/*
 * Attention of packed rows over the paged fp8 cache: sequences with any numbers of new tokens in one launch (the reference
 * runs one-token and prompt rows apart, model/kernels/decode.cu:567-675, 1041-1051). Sequence b's new tokens are rows
 * cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of q and out (bf16 [rows][Hq][128]; cu_seqlens int32 [B + 1], as
 * nc_pages_extend makes it), the last of its seq_lens[b] tokens, all already in the cache; the row at position p attends
 * keys [max(p - window, 0), p] (window < 0: all), scores (q . k) * sm_scale, fp32 softmax (a probability times its key's V
 * scale is rounded to bf16 for its product with V, as in the other attention entries), out bf16. A sequence longer than
 * max_seq_len (<= max_pages * 16) or shorter than its new tokens gets NaN. So does a row that attends keys behind a
 * block-table entry outside [0, num_pages), and with it any rows of its sequence that one wave computes beside it (up to 32
 * (row, head) pairs of a KV head); entries whose keys no row of the sequence attends, such as those behind its window, may
 * hold anything. Rows outside every sequence are left as they are. Row offsets are
 * taken into [0, rows]; if they overlap so that the workspace could not hold the launch, every row gets NaN. A sequence's
 * output bits depend on its own numbers alone, not on the rest of the launch. rows <= 2^24, B <= 1024, Hq / Hkv <= 16.
 */
int nc_packed_attn_fp8(const void *q, const void *k_pages, const void *v_pages, const float *kv_scale,
                       const int32_t *block_table, int max_pages, int num_pages, const int32_t *cu_seqlens,
                       const int32_t *seq_lens, long long rows, int B, int Hq, int Hkv, int max_seq_len, int window,
                       float sm_scale, void *out, void *workspace, size_t workspace_bytes, void *stream);

/*
 * The page bookkeeping of `slots` (<= 4096) sequences over one pool, kept on the device; no counterpart in the reference
 * (its slots own fixed caches, model/kernels/decode.cu:740-763). State: lengths int32 [slots], table int32
 * [slots][max_pages] (-1: no page), free_pages int32 [num_pages] whose first free_count[0] entries are free. arrived: one
 * int32, zero before the first call and left zero by every call. Calls on one state must be ordered. num_pages and
 * max_pages are at most (2^31 - 1) / 16.
 *
 * nc_pages_extend: slot b asks for new_tokens[b] tokens, all or nothing (negative, or past max_pages * 16: none). In slot
 * order, slots get pages while the pool has enough (a slot that needs no page is not refused for pages), then rows while
 * `rows` suffice. The j-th page granted is free_pages[free_count - 1 - j]. Slot b's tokens become rows cu_seqlens[b] ..
 * cu_seqlens[b + 1] - 1 (cu_seqlens int32 [slots + 1]) at positions lengths[b] ..; positions, slot_map int32 [rows]: a
 * row's position and its cache slot 16 page + position % 16, both -1 past the last row; granted int32 [slots]. lengths,
 * table and free_count are updated. No output may overlap new_tokens.
 *
 * nc_pages_trim: slot b longer than keep[b] >= 0 falls back to keep[b] tokens; the pages past them leave the table (-1)
 * and join the free list, the first of them (in slot, then page order) topmost.
 */
int nc_pages_extend(const int32_t *new_tokens, int slots, int32_t *lengths, int32_t *table, int max_pages,
                    const int32_t *free_pages, int32_t *free_count, int num_pages, int rows, int32_t *cu_seqlens,
                    int32_t *positions, int32_t *slot_map, int32_t *granted, int32_t *arrived, void *stream);
int nc_pages_trim(const int32_t *keep, int slots, int32_t *lengths, int32_t *table, int max_pages, int32_t *free_pages,
                  int32_t *free_count, int num_pages, int32_t *arrived, void *stream);

/* Workspace bytes nc_sample_tokens needs for these sizes, at most 7 MB (0 for unsupported sizes). Its first 64 KiB (or all
 * of it, if smaller) are zero-filled before its first call; it is then passed to calls ordered on one stream, of any sizes
 * that it suffices for. It serves no other function. One that is too small or not 16-byte aligned gives NC_ERR_SHAPE. */
size_t nc_sample_workspace_bytes(long long rows, int vocab);

/*
 * A token a row from its logits and one given uniform number: the token choice of a decoding step (reference
 * model/kernels/decode.cu:170-229, 361-411) for callers with logits of their own. logits: fp32, or bf16 (is_bf16), `rows`
 * rows of `vocab` (<= 2^24) at row_stride elements. Per row: temperature fp32 (not above 0: the largest logit, the lowest
 * index among equals); top_k int32, top_p and min_p fp32 (each may be NULL: off); mask (NULL, or uint32 words at
 * mask_stride words a row: token t is allowed where bit t % 32 of word t / 32 is set). With w_i = exp((z_i - max z) /
 * temperature) over the allowed tokens whose logit is neither NaN nor -inf (with a +inf logit only those weigh anything):
 * the top_k largest stay (the lower index first among equals; top_k <= 0: all), of those the tokens with less than top_p
 * of their weight strictly above them (at least the largest; top_p >= 1 or NaN: all), of those the ones with w_i >= min_p
 * (taken into [0, 1]); tokens[row] is the first, in index order, whose running weight exceeds uniform[row] (in [0, 1),
 * else the nearer end; NaN: 0) times the weight of all that are left; -1 where no token is allowed. Weights are held to
 * 2^-46 of the largest (2^(ceil(log2 vocab) - 62) from 65,537 tokens on): smaller ones are never drawn. The result is
 * reproducible and does not depend on the other rows. Calls on any number of streams may overlap, each with a workspace of
 * its own: no workgroup waits without bound for one that may not have started. rows <= 2^22; no rows launch nothing.
 */
int nc_sample_tokens(const void *logits, int is_bf16, long long row_stride, long long rows, int vocab,
                     const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p,
                     const float *min_p, const uint32_t *mask, long long mask_stride, int32_t *tokens, void *workspace,
                     size_t workspace_bytes, void *stream);

/* For tests and measurement: nc_sample_tokens, the workgroups that share a row looking for one another `patience` times
 * (in [0, 65536]) before they give it up and the last of them does it by itself. The tokens are the same. */
int nc_debug_sample_tokens(const void *logits, int is_bf16, long long row_stride, long long rows, int vocab,
                           const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p,
                           const float *min_p, const uint32_t *mask, long long mask_stride, int32_t *tokens,
                           void *workspace, size_t workspace_bytes, int patience, void *stream);

/*
 * The 8-bit form of matrices, their products, and the training of linear layers from 8-bit checkpoints; no counterpart in the
 * reference, whose linear layers are bf16 (model/ops/linear.py:51-57, 135-144). A matrix is held as OCP e4m3fn codes and one
 * power of two for each block, a byte holding its exponent + 127 (e8m0): blocks of 128 columns of a row for activations and
 * gradients, 128 x 128 for weights (the last of a row or column may be shorter). The scale is the least power of two s with
 * max |x| <= 448 s, at least 2^-126 (1 for a block of zeros); a code is x / s rounded to nearest even and stands for code * s. A
 * block that holds an infinity or a NaN becomes NaN (byte 255, codes 0x7F). Columns are a multiple of 16. Codes are dense and
 * 16-byte aligned; scales have rows at a stride in bytes that is a multiple of 4, 4-byte aligned, each row's readable up to a multiple
 * of 4 (the last row's too, but not to the end of its stride).
 */

/* The 8-bit form of rows of activations: x bf16 or fp32 (is_f32) [rows][cols] at row_stride elements (any alignment of its
 * type; 16-byte rows are read faster) -> codes [rows][cols], scale [rows][ceil(cols / 128)] at scale_stride bytes. rows *
 * ceil(cols / 128) < 2^31. */
int nc_fp8_quantize_rows(const void *x, int is_f32, long long row_stride, long long rows, int cols, void *codes, void *scale,
                         long long scale_stride, void *stream);

/* The 8-bit form of a weight: w bf16 or fp32 [n][k] at row_stride elements -> codes [n][k], scale [ceil(n / 128)][ceil(k /
 * 128)], and, unless codes_t is NULL, those of its transpose: codes_t [k][n], scale_t [ceil(k / 128)][ceil(n / 128)] (n then a
 * multiple of 16). n, k <= 2^20. */
int nc_fp8_quantize_weight(const void *w, int is_f32, long long row_stride, int n, int k, void *codes, void *scale,
                           int scale_stride, void *codes_t, void *scale_t, int scale_t_stride, void *stream);

/* out[m][n] = sum_k a[m][k] w[n][k], a [rows][k] and w [n][k] in the 8-bit form, n and k multiples of 16:
 * nc_fp8_matmul         out bf16 [rows][n]
 * nc_fp8_matmul_relu2   relu(out)^2 of the fp32 sums in the 8-bit form: codes [rows][n], scale at scale_stride
 * nc_fp8_matmul_relu2_fast  the same from sums that drop bits where the rows are many, in 0.55 to 0.6 of the time there
 * nc_fp8_matmul_relu2_bwd  out = bf16(sum * 2 sqrt(act)), act [rows][n] in the 8-bit form (as nc_fp8_matmul_relu2 leaves it), and
 *                       the 8-bit form of out: the gradient before a ReLU^2 whose result act is, from the one behind it
 * Sums are fp32, of exact products in nc_fp8_matmul_relu2. In the others they are so but for the eight products of adjacent k that
 * the matrix cores add at a time: of those, bits below 2^-13 of the largest are dropped (at most 2^-10 of the sum of magnitudes, and
 * 1e-5 to 3e-5 of a result as a rule); nc_fp8_matmul_relu2_fast drops none where ceil(rows / 64) ceil(n / 128) is at most the device's
 * number of CUs. The outputs may not overlap the inputs. */
int nc_fp8_matmul(const void *a, const void *a_scale, long long a_scale_stride, const void *w, const void *w_scale,
                  int w_scale_stride, long long rows, int n, int k, void *out, void *stream);
int nc_fp8_matmul_relu2(const void *a, const void *a_scale, long long a_scale_stride, const void *w, const void *w_scale,
                        int w_scale_stride, long long rows, int n, int k, void *codes, void *scale, long long scale_stride,
                        void *stream);
int nc_fp8_matmul_relu2_fast(const void *a, const void *a_scale, long long a_scale_stride, const void *w, const void *w_scale,
                              int w_scale_stride, long long rows, int n, int k, void *codes, void *scale, long long scale_stride,
                              void *stream);
int nc_fp8_matmul_relu2_bwd(const void *a, const void *a_scale, long long a_scale_stride, const void *w, const void *w_scale,
                            int w_scale_stride, long long rows, int n, int k, const void *act, const void *act_scale,
                            long long act_scale_stride, void *out, void *codes, void *scale, long long scale_stride,
                            void *stream);

/* A layer, out = x8 w^T, and a ReLU^2 MLP, out = a8 proj^T with a = relu(x8 fc^T)^2, for serving: x8, a8 the 8-bit forms of x's
 * rows (bf16, or fp32 for a layer with is_f32; [rows][k] at row_stride elements, any alignment of its type) and of the squares of the
 * fp32 sums, w [n][k], fc [hidden][c] and proj [n][hidden] held in 8 bits, out bf16 [rows][n], all widths multiples of 16 up to 2^20.
 * A few rows are bound by reading the weights once; up to 64 that can be read 16 bytes at a time, where they are short and the
 * outputs few enough, are one launch a product. workspace: nc_fp8_*_workspace_bytes (-1 for unsupported sizes; of a layer, for the x
 * and row_stride of the call, and 0 where none is read: it may then be NULL), 16-byte aligned, need not be cleared. A call's workspace
 * is its own until it has run. nc_fp8_mlp_fast is nc_fp8_mlp by way of nc_fp8_matmul_relu2_fast. */
long long nc_fp8_linear_workspace_bytes(const void *x, int is_f32, long long row_stride, long long rows, int n, int k);
int nc_fp8_linear(const void *x, int is_f32, long long row_stride, const void *w, const void *w_scale, int w_scale_stride,
                  long long rows, int n, int k, void *out, void *workspace, long long workspace_bytes, void *stream);
long long nc_fp8_mlp_workspace_bytes(long long rows, int c, int hidden);
int nc_fp8_mlp(const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride, const void *proj,
               const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden, int n, void *out,
               void *workspace, long long workspace_bytes, void *stream);
int nc_fp8_mlp_fast(const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride, const void *proj,
                     const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden, int n, void *out,
                     void *workspace, long long workspace_bytes, void *stream);

/* The gradient of a weight from the 8-bit checkpoint of its layer's input: out[i][j] = sum_m dy[m][i] x[m][j], dy bf16
 * [rows][n1] dense (n1 a multiple of 8), x [rows][n2] in the 8-bit form (scale_stride <= n2). mode 0: out fp32; 1: added to out,
 * fp32; 2: out bf16. Products are exact and sums fp32, in an order that depends on the sizes alone. rows < 2^31, n1 and n2 <=
 * 65,536; rows = 0 launches nothing (and leaves out as it is). workspace: nc_fp8_weight_grad_workspace_bytes (-1 for
 * unsupported sizes), 16-byte aligned, need not be cleared. */
long long nc_fp8_weight_grad_workspace_bytes(long long rows, int n1, int n2);
int nc_fp8_weight_grad(const void *dy, const void *codes, const void *scale, long long scale_stride, long long rows, int n1,
                       int n2, int mode, void *out, void *workspace, long long workspace_bytes, void *stream);

/*
 * The training of a layer and of a ReLU^2 MLP, a direction a call, from the parts above. All in the 8-bit form are at strides as
 * there; rows bf16 at row_stride elements; all widths are multiples of 16.
 *   forward   codes, scale = x in the 8-bit form: the checkpoint; linear: out = it w^T; mlp: act, act_scale = relu(it fc^T)^2 in the
 *             8-bit form, the second checkpoint, and out = it proj^T (_fast: by way of nc_fp8_matmul_relu2_fast)
 *   backward  dy bf16 [rows][n] (dense, 16-byte aligned, where a weight gradient reads it) -> dx bf16 [rows][k] (not wanted where
 *             NULL), from the weights' transposes in the 8-bit form, and dw in nc_fp8_weight_grad's mode, or -1 where it is not wanted:
 *             dx = dy8 w8, dw = dy^T x8; dh = bf16((dy8 p8) 2 sqrt(a8)), dx = dh8 f8, dfc = dh^T x8, dproj = dy^T a8. rows = 0
 *             launches nothing and leaves all outputs as they are.
 * workspace: nc_fp8_*_bwd_workspace_bytes (-1 for unsupported arguments), 16-byte aligned, need not be cleared.
 */
int nc_fp8_linear_fwd(const void *x, long long row_stride, const void *w, const void *w_scale, int w_scale_stride, long long rows,
                      int n, int k, void *codes, void *scale, long long scale_stride, void *out, void *stream);
long long nc_fp8_linear_bwd_workspace_bytes(long long rows, int n, int k, int need_x, int mode);
int nc_fp8_linear_bwd(const void *dy, long long row_stride, const void *codes, const void *scale, long long scale_stride,
                      const void *codes_t, const void *scale_t, int scale_t_stride, long long rows, int n, int k, void *dx,
                      void *dw, int mode, void *workspace, long long workspace_bytes, void *stream);
int nc_fp8_mlp_fwd(const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride,
                   const void *proj, const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden, int n,
                   void *codes, void *scale, long long scale_stride, void *act, void *act_scale, long long act_scale_stride,
                   void *out, void *stream);
int nc_fp8_mlp_fwd_fast(const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride,
                         const void *proj, const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden, int n,
                         void *codes, void *scale, long long scale_stride, void *act, void *act_scale, long long act_scale_stride,
                         void *out, void *stream);
long long nc_fp8_mlp_bwd_workspace_bytes(long long rows, int c, int hidden, int n, int need_x, int fc_mode, int proj_mode);
int nc_fp8_mlp_bwd(const void *dy, long long row_stride, const void *codes, const void *scale, long long scale_stride,
                   const void *act, const void *act_scale, long long act_scale_stride, const void *fc_codes_t,
                   const void *fc_scale_t, int fc_scale_t_stride, const void *proj_codes_t, const void *proj_scale_t,
                   int proj_scale_t_stride, long long rows, int c, int hidden, int n, void *dx, void *dfc, int fc_mode,
                   void *dproj, int proj_mode, void *workspace, long long workspace_bytes, void *stream);

/*
 * Measurement only; no counterpart in the reference. Reads n pages of 2 KiB (one (page, head) of K or V codes) from
 * src (src_bytes, a multiple of 2,048), page order[i] as the i-th (order NULL: page i; an entry outside the buffer
 * reads page 0), with `grid` workgroups of 256 threads, and writes one checksum word per thread to sink
 * (grid x 256 uint32: their XOR is the XOR of every dword read). Its duration is the read-only ceiling of the decode
 * step's page stream. Returns 0, NC_ERR_NULL or NC_ERR_SHAPE (grid outside [1, 65535]).
 */
int nc_debug_read_pages(const void *src, long long src_bytes, const int32_t *order, int n, int grid, uint32_t *sink,
                        void *stream);

#ifdef __cplusplus
}
#endif

#endif /* NANOCHAT_AMD_H */
