/*
 * aspidagpu.h -- C ABI of libaspidagpu.so, the MI355X (gfx950) implementation
 * of Aspida's quantized-weight GPU path.
 *
 * Weight kinds are LLM_Weight.Kind_Code's (src/llm/llm_weight.adb:277-292):
 *   0 = Q4_K (144 B / 256), 1 = Q6_K (210 B), 2 = Q5_K (176 B),
 *   3 = Q3_K (110 B), 4 = Q2_K (84 B), 5 = Q8_0 (8 x 34 B per 256 elements).
 * A weight is row-major [out_dim][in_dim / 256 super-blocks] (GGUF ne0 =
 * in_dim, ne1 = out_dim); activations are contiguous f32, batched ones
 * [batch][in_dim] / [batch][out_dim].  `long` is 64-bit (LP64), Ada's
 * Interfaces.C.long.
 *
 * Host-pointer entry points (the reference ABI) are synchronous and
 * thread-safe.  Weights are mirrored into HBM on first use, keyed by host
 * pointer; the caller must call aspida_gpu_free_weight(w) before freeing or
 * reusing the host bytes of w, and must not free a weight while another
 * thread's call is using it.  On invalid arguments or a HIP failure the
 * output is filled with quiet NaN, a line is printed to stderr and the
 * calling thread's aspida_gpu_last_error() becomes non-zero.
 */
#ifndef ASPIDAGPU_H
#define ASPIDAGPU_H

#ifdef __cplusplus
extern "C" {
#endif

/* ---- reference ABI (symbols resolved by src/llm/llm_gpu.adb:100-146 and
 *      src/llm/llm_qwen_gpu.adb:257-266, 340) ------------------------------ */

/* y[out_dim] = W x.  Replaces gpu/gpu_matvec.cu:502-530.  in_dim must be a
 * multiple of 256 and wbytes >= out_dim * (in_dim / 256) * block bytes.
 * Kind 4 runs Q2_K and kind 5 Q8_0 (the reference sent every kind >= 4 to
 * its Q2_K kernel). */
void aspida_gpu_matvec(const void *w, long wbytes, int kind, int in_dim, int out_dim,
                       const float *x, float *y);

/* Y[batch][out_dim] = X[batch][in_dim] W^T.  Replaces gpu/gpu_matvec.cu:534-553;
 * any batch >= 1 is served (the reference clamped batch to 32); batch < 1 is a
 * no-op as in the reference. */
void aspida_gpu_matmul(const void *w, long wbytes, int kind, int in_dim, int out_dim, int batch,
                       const float *x, float *y);

/* y = W x for a dense row-major f32 W [out_dim][in_dim] (e.g. the f32 MoE
 * router).  Replaces gpu/gpu_matvec.cu:925-935. */
void aspida_gpu_dense_matvec(const void *w, long wbytes, int in_dim, int out_dim,
                             const float *x, float *y);

/* Drop the HBM mirror of host weight w; idempotent, a no-op for unknown w.
 * Replaces gpu/gpu_matvec.cu:494-500. */
void aspida_gpu_free_weight(const void *w);

/* Routed + shared expert FFN of one MoE layer for one token, routing supplied
 * by the caller: y = sum_k top_w[k] * Down_e(silu(Gate_e x) * Up_e x)
 * (e = top_idx[k], 0-based, ascending k) + g * SharedDown(silu(SharedGate x)
 * * SharedUp x), g = sigmoid(shared_gate_inp . x) when gate_inp_len > 1 and
 * shared_gate_inp is non-null, else 1.  Routed expert tensors are
 * [n_exp][rows][cols] with bytes / n_exp per expert.  Replaces
 * gpu/gpu_matvec.cu:1673-1758; top_k may be up to 32 (the reference silently
 * truncated it to 8); dim and intermed must be multiples of 256.  When gate,
 * up, shared gate and shared up share one kind and down and shared down
 * another, the experts are mirrored in the packed layout and run by the
 * grouped kernels of aspida_moe_experts_packed_dev. */
void aspida_gpu_moe_experts(const float *x, int dim, int top_k, int intermed, int n_exp,
                            const int *top_idx, const float *top_w,
                            const void *gate_w, long gate_bytes, int gate_kind,
                            const void *up_w, long up_bytes, int up_kind,
                            const void *down_w, long down_bytes, int down_kind,
                            const void *shg_w, long shg_bytes, int shg_kind,
                            const void *shu_w, long shu_bytes, int shu_kind,
                            const void *shd_w, long shd_bytes, int shd_kind,
                            const float *shared_gate_inp, int gate_inp_len, float *y);

/* Return and clear the calling thread's last error (0 = none).  Same
 * signature and "return and clear" contract as gpu/gpu_matvec.cu:2348-2352. */
int aspida_gpu_last_error(void);

/* ---- device-pointer entry points (no counterpart in the reference ABI: for
 *      callers whose weights and activations already live in HBM, e.g. a
 *      resident decode chain).  Asynchronous on `stream` (a hipStream_t, NULL =
 *      null stream); return 0 or a negative errno / positive hipError_t. ---- */

/* xq[r][i] = sum of x[r][16 i .. 16 i + 15], r < rows: the per-group
 * activation sums the K-quant kernels take (in_dim % 16 == 0). */
int aspida_kq_xsum_dev(const float *x, int in_dim, int rows, float *xq, void *stream);

/* Device form of aspida_gpu_matvec; xq from aspida_kq_xsum_dev(x). */
int aspida_kq_matvec_dev(int kind, const void *w, int in_dim, int out_dim, const float *x,
                         const float *xq, float *y, void *stream);

/* Lane-interleaved ("packed") layout of the batch-1 decode kernels: tiles of
 * 64 rows, each tile's super-block column stored as 16-byte chunk planes with
 * one chunk per row, so a wave reads 1 KB per load and each lane owns one
 * row.  Same bytes as the ggml layout, regrouped (rows past out_dim in the
 * last tile are zero).  The same math as QMatVec
 * (src/llm/llm_dequant.adb:808-932) and the reference's batch-1 kernels
 * (gpu/gpu_matvec.cu:149-383), over a layout of this library's own.
 * aspida_kq_packed_bytes: size of the packed image (0 for a bad kind/shape).
 * aspida_kq_pack_dev / aspida_kq_unpack_dev: ggml <-> packed, on `stream`. */
long long aspida_kq_packed_bytes(int kind, int in_dim, int out_dim);
int aspida_kq_pack_dev(int kind, const void *w, int in_dim, int out_dim, void *packed, void *stream);
int aspida_kq_unpack_dev(int kind, const void *packed, int in_dim, int out_dim, void *w, void *stream);

/* Launch split aspida_kq_matvec_packed_dev uses for this shape: waves per
 * workgroup (the kernel is kq_mv_packed<kind, waves>), workgroups per 64-row
 * tile and super-block columns per wave (their product is in_dim / 256). */
/* The kernel and split aspida_kq_matvec_packed_dev uses for a kind and shape
 * under the current engine (aspida_kq_set_mv_engine): returns 1 for the
 * matrix-core kernel on 64-row workgroups kq_mv_mfma<kind, waves, walk> (walk
 * 0: one column per wave, 1: prefetching columns), 2 for the same kernel
 * taking its columns one after another (walk 2), 3 and 4 for the same two
 * walks of the 16-row-workgroup kernel kq_mv_mfma16<kind, waves, walk>
 * (groups_per_tile is then 1), 0 for the vector kernel
 * kq_mv_packed<kind, waves, prefetch>, or -EINVAL.  No reference counterpart. */
int aspida_kq_matvec_plan(int kind, int in_dim, int out_dim, int *waves_per_group, int *groups_per_tile,
                          int *columns_per_wave);
int aspida_kq_packed_plan(int in_dim, int out_dim, int *waves_per_group, int *groups_per_tile,
                          int *columns_per_wave);

/* y[out_dim] = W x for packed W: the batch-1 decode path.  Per-group
 * activation sums are formed inside the kernel (no xq).  x must be 16-byte
 * aligned.  The library keeps a small workspace per stream (allocated on the
 * first call for a stream and shape, so warm up before graph capture);
 * calls on one stream are ordered, calls on different streams are
 * independent. */
int aspida_kq_matvec_packed_dev(int kind, const void *packed, int in_dim, int out_dim, const float *x,
                                float *y, void *stream);

/* Allocation-free form of aspida_kq_matvec_packed_dev: same kernels, launch
 * split and results (bit for bit), but the workspace -- per-tile arrival
 * counters and cross-workgroup partial sums -- lives in a fixed device array
 * of this library (6 MiB, one copy per GPU, held until the process ends), so
 * the call never allocates device memory: no hipMalloc, hipFree or allocating
 * library routine.  No counterpart in the reference.  For callers that cannot
 * allocate: code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc.  Limit: out_dim up to 262,144 rows and at most 1,310,720
 * partial sums (tiles x workgroups per tile x 64); larger shapes return
 * -E2BIG and launch nothing.  Every call on one GPU shares the array, so calls
 * that overlap in time on one GPU (different streams or threads) race and
 * give wrong results: order them on one stream.  x must be 16-byte aligned. */
int aspida_kq_matvec_packed_noalloc_dev(int kind, const void *packed, int in_dim, int out_dim, const float *x,
                                        float *y, void *stream);

/* y_a = A x and y_b = B x for two packed matrices that share the input (e.g.
 * the q|k and v projections of a decoder layer), in one launch for the kind
 * pairs (Q4_K, Q6_K), (Q5_K, Q6_K) and equal kinds Q4_K, Q5_K, Q6_K, Q8_0;
 * other pairs run as two launches.  Same results as two calls of
 * aspida_kq_matvec_packed_dev. */
int aspida_kq_matvec2_packed_dev(int kind_a, const void *packed_a, int out_a, float *y_a, int kind_b,
                                 const void *packed_b, int out_b, float *y_b, int in_dim, const float *x,
                                 void *stream);

/* Y[batch][out_dim] = X[batch][in_dim] W^T for packed W: any batch.  Products
 * run on MFMA (activations split into f16 hi + lo, exact integer codes, f32
 * scales), up to 512 vectors per weight pass, except few vectors of Q5_K,
 * Q3_K, Q2_K and Q8_0 (up to 4 to 7 by shape, 24 on the smallest matrices),
 * which run on the vector kernel, each row bit-identical to
 * aspida_kq_matvec_packed_dev on it (aspida_kq_set_mv_engine(1)).  A row's
 * bits otherwise depend on how many vectors the product has; while that
 * override is set, these four kinds run there for any batch.
 * x must be 16-byte aligned; workspace as for aspida_kq_matvec_packed_dev
 * (sized by in_dim and out_dim, the many-vector part for any batch).
 * The same math as the reference's batched kernels (gpu/gpu_matvec.cu:234-382)
 * without its batch limit of 32. */
int aspida_kq_matmul_packed_dev(int kind, const void *packed, int in_dim, int out_dim, int batch,
                                const float *x, float *y, void *stream);

/* Device form of aspida_gpu_matmul; xq from aspida_kq_xsum_dev(x, .., batch). */
int aspida_kq_matmul_dev(int kind, const void *w, int in_dim, int out_dim, int batch,
                         const float *x, const float *xq, float *y, void *stream);

/* Small-batch product forced onto the vector-ALU kernels (the reference
 * numerics path the MFMA kernels are checked against). */
int aspida_kq_matmul_valu_dev(int kind, const void *w, int in_dim, int out_dim, int batch,
                              const float *x, const float *xq, float *y, void *stream);

/* dst[out_dim][in_dim] = dequantized W, bit-identical to the CPU decoders
 * Decode_Q*K_Block (src/llm/llm_dequant.adb:122-554) and Dequant_Q8_0
 * (606-630), including their Inf/NaN -> +0.0 reading of f16 scales. */
int aspida_kq_dequant_dev(int kind, const void *w, int in_dim, int out_dim, float *dst, void *stream);

/* Device form of aspida_gpu_dense_matvec. */
int aspida_dense_matvec_dev(const float *w, int in_dim, int out_dim, const float *x, float *y,
                            void *stream);

/* MoE router for T tokens: logits[t][e] = router_w[e][:] . x[t][:] (f32,
 * [n_exp][dim]), stable softmax, greedy top-k (strict >, lowest index wins
 * ties), renormalised weights (src/llm/llm_moe.adb:136-197).  Writes
 * logits[T][n_exp], top_idx[T][top_k] (0-based) and top_w[T][top_k].
 * n_exp <= 1024, top_k <= 32, dim % 4 == 0, router_w and x 16-byte aligned.
 * Uses the stream's workspace like aspida_kq_matvec_packed_dev (allocated on
 * the first call for a stream and T, so warm up before graph capture). */
int aspida_moe_route_dev(const float *router_w, int n_exp, int dim, int T, int top_k, const float *x,
                         float *logits, int *top_idx, float *top_w, void *stream);

/* Floats of `work` aspida_moe_experts_dev needs. */
long aspida_moe_work_floats(int T, int dim, int top_k, int intermed);

/* Device form of aspida_gpu_moe_experts for T tokens: x [T][dim], top_idx /
 * top_w [T][top_k], y [T][dim]; routed expert e of a projection starts at
 * byte e * *_stride of its tensor; shared_gate_inp may be NULL (ungated). */
int aspida_moe_experts_dev(const float *x, int T, int dim, int top_k, int intermed, int n_exp,
                           const int *top_idx, const float *top_w,
                           const void *gate_w, long gate_stride, int gate_kind,
                           const void *up_w, long up_stride, int up_kind,
                           const void *down_w, long down_stride, int down_kind,
                           const void *shg_w, int shg_kind, const void *shu_w, int shu_kind,
                           const void *shd_w, int shd_kind, const float *shared_gate_inp,
                           float *work, float *y, void *stream);

/* Grouped MoE over packed experts.  Same arithmetic contract as
 * aspida_moe_experts_dev (LLM_MoE.Forward steps 4-5,
 * src/llm/llm_moe.adb:249-299; the reference shim's moe_experts,
 * gpu/gpu_matvec.cu:1673-1760), but the expert matrices are in the packed
 * layout (aspida_moe_pack_experts_dev) and each expert's weights are read once
 * per launch however many of the T tokens chose it.  Gate, up, shared gate
 * and shared up are of kind gu_kind, down and shared down of down_kind.
 * dim and intermed multiples of 256, top_k <= 32.  x 16-byte aligned, work
 * 256-byte aligned with aspida_moe_packed_work_bytes bytes.  Deterministic:
 * each y[t] sums its slots in ascending k, shared expert last.  top_idx
 * entries outside [0, n_exp) leave that token's y unwritten. */
long aspida_moe_packed_work_bytes(int T, int dim, int intermed, int top_k);
int aspida_moe_pack_experts_dev(int kind, const void *src, long src_stride, int in_dim, int out_dim, int n,
                                void *dst, void *stream);
int aspida_moe_experts_packed_dev(const float *x, int T, int dim, int top_k, int intermed, int n_exp,
                                  const int *top_idx, const float *top_w, const void *gate_p,
                                  const void *up_p, int gu_kind, const void *down_p, int down_kind,
                                  const void *shg_p, const void *shu_p, const void *shd_p,
                                  const float *shared_gate_inp, void *work, float *y, void *stream);

/* ---- rotary positions and the 4-bit key/value cache ---------------------------
 * What a decoder layer does between its q|k|v and its output product, on
 * device pointers.  No counterpart in the reference ABI, whose attention lives
 * behind its resident chain (gpu/gpu_matvec.cu:2063-2141).
 * Activation types: 0 = f32, 1 = f16, 2 = bf16; operands need the alignment
 * of their type only, and rows lie `stride` elements apart (at least heads *
 * head_dim, which are contiguous).  Sums, softmax statistics and lse are f32.
 * The calls allocate nothing, keep nothing and may be captured into a graph
 * (its replays read the device arrays anew: lengths, row starts, tables). */

/* A rotation: pair i of a head's first rot_dim values (even, 2 to 256) turns
 * by pos * f_i, f_i = base^(-2 i / rot_dim); the angle is formed in f64.
 * After freq_factors and scaling f_i must be at most 2^19.
 * Pairs are (i, i + rot_dim / 2), or (2 i, 2 i + 1) when interleaved; the
 * values behind rot_dim pass through.  freq_factors (host, rot_dim / 2 values
 * as in a GGUF rope_freqs.weight, or NULL) divide f first.  scaling:
 *   0 none;
 *   1 linear: f / factor;
 *   2 bands: f / factor for pairs that turn fewer than `low` times over
 *     `context` positions, f for those that turn more than `high` times, and
 *     a blend linear in the turns between;
 *   3 blend by pair (YaRN): f / factor from the pair that turns `low` times on,
 *     f up to the one that turns `high` times, linear in the pair between;
 *     the rotated values are also multiplied by 0.1 ln(factor) + 1.
 * magnitude, when not 0, replaces that multiplier (1 for the other scalings).
 * aspida_rope_create returns a handle (host memory only; NULL and
 * aspida_gpu_last_error on bad parameters); aspida_rope_table copies its
 * rot_dim / 2 frequencies and multiplier out. */
typedef struct aspida_rope_params {
  int rot_dim, interleaved, scaling, reserved;
  double base, factor, low, high, context, magnitude;
  const float *freq_factors;
} aspida_rope_params;
void *aspida_rope_create(const aspida_rope_params *params);
int aspida_rope_table(const void *rope, double *freq, double *magnitude);
void aspida_rope_destroy(void *rope);

/* y = x [n_tok][n_heads][head_dim] with every head rotated to its token's
 * pos[n_tok] (any int); y may be x with the same stride, else they must not
 * overlap.  inverse != 0 turns back: with magnitude 1 that undoes the
 * rotation, and in general it is the gradient (y = dL/dx of x = dL/dy).
 * -ENOTSUP for heads of more than 256 of the widest pieces (16 bytes, two
 * values, one) that divide their runs. */
int aspida_rope_dev(const void *rope, int type, const void *x, long long x_stride, int n_tok, int n_heads,
                    int head_dim, const int *pos, int inverse, void *y, long long y_stride, void *stream);

/* The cache of one layer: pages of 64 slots, each aspida_kv4_page_bytes long
 * (80 head_dim per kv head: 5 bits a value), and per sequence a row of
 * max_pages page ids; slot j of sequence b is in page table[b][j / 64].  A
 * sequence's token t is at slot t, until an eviction.  head_dim is 64, 128 or
 * 256.  Every 32 values x of a token's head keep m = f16(min x), a step d
 * ((max x - m) / 15 rounded up to 7 significant bits, f16) and 4-bit codes q,
 * the integers nearest (x - m) / d (ties to even): a code stands for
 * d q + m.  A token whose key or value in some kv head has a group with a
 * value that is not finite, a minimum beyond f16 or a step above 254 reads
 * back as NaN there, key and value, and a row that sees it comes out as NaN.
 * Page ids outside [0, n_pages) and slots past max_pages name no memory:
 * appends to them are dropped, reads give NaN, and a row that sees such a slot
 * comes out as NaN.  No two table entries that a call writes to may name the
 * same page.  pages is 16-byte aligned. */
typedef struct aspida_kv4 {
  int head_dim, n_kv, n_pages, max_pages;
  void *pages;       /* device, n_pages * aspida_kv4_page_bytes(head_dim, n_kv) */
  const int *table;  /* device, [n_seq][max_pages] */
} aspida_kv4;
long long aspida_kv4_page_bytes(int head_dim, int n_kv);

/* Rows of new tokens, in the calls below: sequence b has rows row_start[b] ..
 * row_start[b + 1] - 1 (device, n_seq + 1 ascending values up to n_rows; NULL:
 * one row each, n_rows = n_seq).  kv_len[b] (device) is its length with them:
 * its n rows are the tokens at slots kv_len[b] - n .. kv_len[b] - 1, those
 * below 0 being left out.  Rows past the last sequence are not touched.  At
 * most 65535 sequences; 0 rows or sequences are a no-op. */

/* Writes k and v rows [n_rows][n_kv][head_dim] into the cache.  With a rope
 * (rot_dim <= head_dim) keys are rotated to pos[n_rows] first, in f64 and
 * rounded to f32 once; NULL stores them as they are. */
int aspida_kv4_append_dev(const aspida_kv4 *cache, int type, const void *k, long long k_stride, const void *v,
                          long long v_stride, int n_rows, int n_seq, const int *row_start, const int *kv_len,
                          const void *rope, const int *pos, void *stream);

/* The values the cache stands for, at the slots of such rows. */
int aspida_kv4_read_dev(const aspida_kv4 *cache, int type, int n_rows, int n_seq, const int *row_start,
                        const int *kv_len, void *k, long long k_stride, void *v, long long v_stride, void *stream);

/* out[row][h] = sum_j softmax_j(scale * q[row][h] . k_j) v_j for q rows
 * [n_rows][n_heads][head_dim] that are already in the cache: the row at slot
 * p sees slots j <= p, and with window > 0 only j > p - window.  Query heads
 * h * n_kv / n_heads share kv heads (n_heads a multiple of n_kv).  lse (NULL
 * or [n_rows][n_heads]) receives log sum_j exp(scale * q . k_j).  A row that
 * sees nothing (kv_len 0, or a slot below 0) gets 0, and lse -inf; what masked
 * slots hold never matters.  max_rows: at least the rows of the longest
 * sequence (what a sequence has past it comes out as NaN).  work: 256-byte
 * aligned, aspida_kv4_attn_work_bytes long: 6 to 9 MB, the same for all calls
 * of a head_dim, so one workspace serves them in turn; launches that share it
 * must be ordered.  out must not overlap q. */
long long aspida_kv4_attn_work_bytes(const aspida_kv4 *cache, int n_heads, int n_rows, int n_seq, int max_rows);
int aspida_kv4_attn_dev(const aspida_kv4 *cache, int type, const void *q, long long q_stride, int n_heads, int n_rows,
                        int n_seq, const int *row_start, int max_rows, const int *kv_len, float scale, int window,
                        void *out, long long out_stride, float *lse, void *work, void *stream);

/* The attention weight that each slot receives from such rows, given their
 * lse: acc_out[b][g][j] = acc_in[b][g][j] + the sum over b's rows that see j
 * and the query heads of kv head g of exp(scale * q . k_j - lse), nothing for
 * slots from kv_len[b] on; both [n_seq][n_kv][acc_stride], slots past
 * acc_stride being left out.  acc_in may be acc_out, or NULL for zeros.
 * max_rows: at least the rows of the longest sequence (one with more gives
 * NaN to the slots it sees).  The same bits every time (no atomics). */
int aspida_kv4_weigh_dev(const aspida_kv4 *cache, int type, const void *q, long long q_stride, int n_heads, int n_rows,
                         int n_seq, const int *row_start, int max_rows, const int *kv_len, float scale, int window,
                         const float *lse, const float *acc_in, float *acc_out, long long acc_stride, void *stream);

/* Shrinks each sequence to `keep` slots, per kv head: of kv_len[b] > keep
 * slots the first `first` and the last `recent` stay, and of the others the
 * heaviest by acc (NaN, negative and missing weights count as 0), among equals
 * the lowest; they move in order to slots 0 .. keep - 1 of dst's pages (same
 * head_dim and n_kv, its own table, no page in common with what src's table
 * names).  Shorter sequences are copied.  new_len[n_seq] = min(kv_len, keep)
 * (it may be kv_len, for lengths that shrink in place);
 * idx and acc_out [n_seq][n_kv][keep] hold the old slot and weight of each
 * new one, -1 and 0 past new_len.  first + recent <= keep. */
int aspida_kv4_evict_dev(const aspida_kv4 *src, int n_seq, const int *kv_len, const float *acc, long long acc_stride,
                         int keep, int first, int recent, const aspida_kv4 *dst, int *new_len, int *idx,
                         float *acc_out, void *stream);

/* Resident decode chain: an ordered list of packed matvecs (steps) run by ONE
 * persistent launch, with no launch boundary between them -- e.g. every
 * weight matrix of a decoder pass.  A step whose x lies inside an earlier
 * step's y (its producer: the latest earlier step whose y overlaps x; x must
 * lie wholly inside it) waits, per 256-element column, only for the 64-row
 * tiles of the producer that write those elements, while the weight loads
 * of the following columns are already in flight; other steps read x as
 * given.  No step may write memory that an earlier step reads or writes, or
 * its own x.  Same arithmetic per row as aspida_kq_matvec_packed_dev (a
 * different, fixed order of the per-column sums; deterministic).  No
 * counterpart in the reference, whose per-call ABI this path replaces for
 * callers that keep weights and activations in HBM
 * (aspida_gpu_matvec, gpu/gpu_matvec.cu:502-530, called per matrix).
 * aspida_kq_chain_create validates the steps and allocates the chain's
 * flags and partial sums (NULL on error, see aspida_gpu_last_error);
 * aspida_kq_chain_run launches it on `stream` and allocates nothing (runs of
 * one chain must be ordered); aspida_kq_chain_check synchronises and returns
 * 1 if a dependency wait gave up since the last check (outputs of that run
 * unreliable; only when the device could not keep every workgroup
 * resident), else 0; aspida_kq_chain_workgroups: the launch's workgroups. */
typedef struct aspida_kq_step {
  int kind, in_dim, out_dim, reserved;
  const void *packed;   /* aspida_kq_pack_dev layout */
  const float *x;       /* [in_dim], 16-byte aligned */
  float *y;             /* [out_dim] */
} aspida_kq_step;
void *aspida_kq_chain_create(const aspida_kq_step *steps, int nsteps);
int aspida_kq_chain_run(void *chain, void *stream);
int aspida_kq_chain_check(void *chain);
int aspida_kq_chain_workgroups(void *chain);
void aspida_kq_chain_destroy(void *chain);

/* ---- resident model chain (the reference's chain ABI) -----------------------
 * One decode step of a whole MoE model on device-resident weights: the
 * embedding row; per layer nx = RMSNorm(H, attn_norm), H += Mix nx, then
 * nr = RMSNorm(H, post_norm), H += MoE(nr) (LLM_Qwen_Blk.Step,
 * src/llm/llm_qwen_blk.adb:125-170, with LLM_MoE.Forward's router, top-k and
 * experts); then logits = LM RMSNorm(H, final_norm) (src/llm/llm_qwen.adb:
 * 1199-1203).  RMSNorm eps 1e-6.  Weights are given as host pointers and
 * copied into HBM at registration (quantised matrices repacked, a quantised
 * router decoded to f32); the chain owns those copies until
 * aspida_gpu_chain_reset.  The first forward of a lane count runs eagerly;
 * later ones replay a HIP graph captured after it (ASPIDA_NO_GRAPH in the
 * environment, or aspida_kq_chain_set_graphs(0), keeps every forward eager).
 * The reference registers each layer's mixer (attention or delta-net) through
 * aspida_gpu_chain_fattn / aspida_gpu_chain_dnet, which this library does not
 * export: a layer and its mixer -- one matvec -- are registered with
 * aspida_kq_chain_layer instead, so the Ada host's Chain_Available
 * (src/llm/llm_qwen_gpu.adb:554-560) stays false and it keeps its per-layer
 * paths.  Errors: registration failures mark the chain not ready
 * (aspida_gpu_chain_ready() == 0 until a reset); a failed forward fills the
 * logits with NaN; both set aspida_gpu_last_error. */

/* Drop every registered layer and the model.  Replaces gpu/gpu_matvec.cu:2063-2066. */
void aspida_gpu_chain_reset(void);

/* Attach the MoE block to the last registered layer (no-op with no layer).
 * Weight kinds as above (router_k may also be -1: f32 [n_exp][dim]); routed
 * tensors hold n_exp experts of bytes / n_exp each; sgi is the shared-expert
 * gate input when sgi_len > 1 (then sgi_len == dim), else the shared expert is
 * ungated.  n_exp <= 1024, top_k <= 32, intermed % 256 == 0.  Gate, up and
 * the shared gate/up of one kind and both downs of another run on the grouped
 * kernels over packed experts, other mixes on the per-projection kernels.
 * Replaces gpu/gpu_matvec.cu:2143-2199. */
void aspida_gpu_chain_moe(const void *router_w, long router_b, int router_k,
                          const void *gate_w, long gate_b, int gate_k,
                          const void *up_w, long up_b, int up_k,
                          const void *down_w, long down_b, int down_k,
                          const void *shg_w, long shg_b, int shg_k,
                          const void *shu_w, long shu_b, int shu_k,
                          const void *shd_w, long shd_b, int shd_k,
                          const float *sgi, long sgi_b, int sgi_len,
                          int n_exp, int top_k, int intermed);

/* Embedding table (f32 [embed_b / (4 dim)][dim]), final norm (f32 [dim]) and
 * output head ([vocab][dim] of kind lm_k, -1 = f32).  Replaces
 * gpu/gpu_matvec.cu:2201-2211. */
void aspida_gpu_chain_model(const float *embed, long embed_b, const float *fnorm, long fnorm_b,
                            const void *lm, long lm_b, int lm_k, int dim, int vocab);

/* 1 when a model, at least one layer and no failed registration.  Replaces
 * gpu/gpu_matvec.cu:2213. */
int aspida_gpu_chain_ready(void);

/* A generation's start and end: drop the captured graphs.  attn_handles is
 * unused (the matvec mixers keep no per-generation state).  Replace
 * gpu/gpu_matvec.cu:2328-2340. */
void aspida_gpu_chain_begin(const int *attn_handles);
void aspida_gpu_chain_end(void);

/* logits[vocab] of one token whose embedding row is embed_row; pos and
 * attn_handles are unused (see aspida_gpu_chain_begin).  Synchronous.
 * Replaces gpu/gpu_matvec.cu:2356-2400. */
void aspida_gpu_chain_forward(int embed_row, int pos, const int *attn_handles, float *logits);

/* logits[B][vocab] of B lanes (rows[B]) in one step: the matvecs become
 * small-batch products and the MoE blocks run the B tokens together (each
 * expert's weights read once per layer).  1 <= B <= 64 and B * top_k <= 1024;
 * B < 1 is a no-op as in the reference (which clamped B to its lane limit
 * instead of failing).  Replaces gpu/gpu_matvec.cu:2783-2961. */
void aspida_gpu_chain_forward_batch(int B, const int *rows, const int *pos, const int *handles, float *logits);

/* A layer (this library's stand-in for chain_fattn / chain_dnet): attention
 * and post-attention norms (f32 [dim], an_b = pn_b = 4 dim bytes, dim % 256 ==
 * 0) and the mixer, a [dim][dim] matrix of kind mix_k (-1 = f32), or none when
 * mix_w is NULL.  Returns 0 or an error (the chain is then not ready).  No
 * reference counterpart. */
int aspida_kq_chain_layer(const float *attn_norm, long an_b, const float *post_norm, long pn_b,
                          const void *mix_w, long mix_b, int mix_k);

/* The residual stream H[B][dim] after the embedding and the first n_layers
 * layers (0 <= n_layers <= layer count), run eagerly: the chain's state
 * step by step.  Returns 0 or an error.  No reference counterpart. */
int aspida_kq_chain_forward_layers(int B, const int *rows, int n_layers, float *hidden);

/* Graph replay on (1) or off (0) for later forwards; drops captured graphs.
 * aspida_kq_chain_graphs: graphs currently captured.  No reference
 * counterpart. */
int aspida_kq_chain_set_graphs(int on);
int aspida_kq_chain_graphs(void);

/* ---- GGUF tensor layout (host only) ----------------------------------------
 * A reader of GGUF model files for locating and checking real weights: the
 * header, metadata and tensor descriptors with the reference loader's rules
 * (LLM_GGUF.Open_From_Source, src/llm/llm_gguf.adb:317-560; byte sizes per
 * Checked_Byte_Size, 238-258; type codes per To_GGML_Type, 266-291).  A
 * tensor's kind is this library's code (0 Q4_K, 1 Q6_K, 2 Q5_K, 3 Q3_K,
 * 4 Q2_K, 5 Q8_0; LLM_Weight.Kind_Code, src/llm/llm_weight.adb:277-292) or -1;
 * dims[0] is ne0 (in_dim of a weight), dims[1] ne1 (out_dim). */
typedef struct aspida_gguf aspida_gguf;
typedef struct aspida_gguf_tensor_info {
  const char *name;       /* valid until aspida_gguf_close */
  int ggml_type, kind, n_dims;
  long long dims[4];
  long long file_offset;  /* absolute byte offset of the data in the file */
  long long bytes;
} aspida_gguf_tensor_info;
/* NULL on a malformed or unreadable file; aspida_gguf_error() says why. */
aspida_gguf *aspida_gguf_open(const char *path);
const char *aspida_gguf_error(void);
void aspida_gguf_close(aspida_gguf *g);
int aspida_gguf_version(const aspida_gguf *g);
long long aspida_gguf_alignment(const aspida_gguf *g);
long long aspida_gguf_data_start(const aspida_gguf *g);
long long aspida_gguf_tensor_count(const aspida_gguf *g);
long long aspida_gguf_meta_count(const aspida_gguf *g);
/* A metadata value as text (arrays as "[array: N]"), or NULL. */
const char *aspida_gguf_meta(const aspida_gguf *g, const char *key);
/* Index of the tensor named `name`, or -1. */
long long aspida_gguf_find(const aspida_gguf *g, const char *name);
int aspida_gguf_tensor(const aspida_gguf *g, long long i, aspida_gguf_tensor_info *out);
/* Copy tensor i's bytes to dst (cap >= its byte size); returns the byte count
 * or a negative errno. */
long long aspida_gguf_read(const aspida_gguf *g, long long i, void *dst, long long cap);

/* ---- test and tuning hooks (no reference counterpart) ----------------------
 * The aspida_kq_set_* overrides below are per calling thread: each changes
 * the kernel choice of the launches the calling thread makes from then on,
 * and no other thread's.  They exist for tests and tuning runs; production
 * callers leave them at their defaults. */

/* Small-batch workspace check, host only (launches nothing): the bytes of
 * activation split and partial sums the library allocates on a stream for a
 * batched product of this kind, shape and batch (*allocated), and the most any single
 * launch of that product uses (*needed).  Returns 0 or -EINVAL. */
int aspida_kq_matmul_workspace(int kind, int in_dim, int out_dim, int batch, long long *allocated,
                               long long *needed);

/* Split override for the packed kernels (aspida_kq_packed_plan): waves per
 * workgroup (a power of two <= 16) and workgroups per tile, applied to every
 * shape whose in_dim / 256 they divide; 0, 0 restores the built-in choice.
 * Per calling thread; for tuning and tests. */
int aspida_kq_set_packed_plan(int waves_per_group, int groups_per_tile);

/* Engine of the batch-1 packed matvec (aspida_kq_matvec_packed_dev and the
 * calls built on it): 0 = matrix cores (MFMA) for the five K-quants, the vector
 * kernel for Q8_0 (the default); 1 = the vector kernel for every kind, and no
 * many-job MoE or many-vector product.
 * Per calling thread; for comparison and tests.  No reference counterpart.
 * Returns 0, or -EINVAL for another value. */
int aspida_kq_set_mv_engine(int engine);

/* Engine of the packed small-batch product (batch > 1 in
 * aspida_kq_matmul_packed_dev and aspida_gpu_matmul): 0 = the built-in choice
 * (the many-vector kernel wherever it measured ahead: every kind above 64
 * vectors, most matrices above 4 to 16; below that line, Q4_K and Q6_K: up to 4
 * vectors on the batch-1 matrix-core kernel where the batch-1 plan is 16-row workgroups, else the one-pass kernel -- Q6_K
 * keeps the batch-1 kernel at 2 vectors -- then the one-pass kernel up to
 * 16 vectors (on matrices of at least 8192 64-row-by-256-column blocks,
 * such as output heads, the 16-vector matrix-core kernel instead, Q6_K from
 * 5 vectors); above 16 the one-pass kernel for Q6_K -- in launches of 32
 * vectors where it takes 64-row tiles; above 32 vectors on at most 1024
 * such blocks the wave-per-column kernel (6) -- and the 64-vector matrix-core
 * kernel for Q4_K; other kinds on the vector kernel); 1 = the vector kernel; 2 = the 64-vector and 3 = the
 * 16-vector matrix-core kernel; 4 = the one-pass matrix-core kernel (up to
 * 64 vectors per weight pass); 5 = the batch-1 matrix-core kernel on up to 4
 * vectors per launch; 6 = the wave-per-column matrix-core kernel (Q4_K and
 * Q6_K with in_dim a multiple of 1024: one wave per 64-row tile and
 * 256-element column, activations split in a pre-pass); for the kinds that
 * have one (others stay on the vector kernel).
 * Per calling thread; for comparison and tests.  No reference counterpart.
 * Returns 0, or -EINVAL for another value. */
int aspida_kq_set_mm_engine(int engine);

/* Workgroup shape of the matrix-core matvec: 0 = the built-in choice (16-row
 * workgroups over all columns for matrices of up to two such blocks per
 * compute unit, 64-row workgroups above), 1 = 64-row, 2 = 16-row workgroups.
 * Per calling thread; for tuning and tests.  No reference counterpart.
 * Returns 0 or -EINVAL. */
int aspida_kq_set_mfma_rows(int mode);

/* Tuning of the matrix-core matvec's splits with several columns per wave:
 * 0 = the built-in choice, 1 = prefetching waves (two register sets),
 * 2 = columns one after another (one register set, more waves per CU).
 * Per calling thread.  No reference counterpart.  Returns 0 or -EINVAL. */
int aspida_kq_set_mfma_pipeline(int mode);

/* Launch-shape override for batch-1 matvecs: rows per lane group per step
 * (1, 2 or 4) and resident waves launched per CU (1..64); rows_per_wave <= 0
 * restores the built-in choice.  Per calling thread; for tuning and tests. */
int aspida_kq_set_mv_config(int rows_per_wave, int waves_per_cu);

#ifdef __cplusplus
}
#endif
#endif
