/*
 * rdnattention_ext.h -- entry points of librdnattention.so that have no
 * counterpart in the reference's C ABI: paged key/value caches, quantisers,
 * and what testing and measurement need; the four drop-in symbols in
 * rdnattention.h do not depend on them.  Same return-code and error-string conventions as rdnattention.h.
 */
#ifndef RDNATTENTION_EXT_H
#define RDNATTENTION_EXT_H

#include "rdnattention.h"

/* Kernel path for rdna_attention_forward_path(). */
#define RDNA_PATH_AUTO 0    /* what rdna_attention_forward() picks */
#define RDNA_PATH_PREFILL 1 /* tiled prefill kernel */
#define RDNA_PATH_SPLITK 2  /* split-K decode kernel + combine */

/* rdna_attention_forward() with the kernel path forced, so tests can run the
 * prefill and split-K kernels on the same input.  No reference counterpart:
 * for parity tests and benchmarks. */
RDNA_API int32_t rdna_attention_forward_path(
    const void* q, const void* k, const void* v, void* output,
    const void* rot_cos, const void* rot_sin,
    int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
    int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
    int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_s,
    int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s,
    uint32_t batch_size, uint32_t num_heads, uint32_t num_kv_heads,
    uint32_t seq_len, uint32_t key_seq_len, uint32_t head_dim,
    float scale, int32_t causal, int32_t has_rope, int32_t window_size,
    int32_t path, void* hip_stream);

/* Releases the device memory the library keeps for reuse: the scratch
 * buffers (RoPE-rotated K copies, split-K and paged partials, prefixes' parts,
 * quantiser partials, INT8 decode scores) it caches per (device, stream, use), grown to the largest
 * call so far (at most 256 MiB each, at most 1 GiB per device over all
 * streams and uses), the scratch of captured graphs that have been destroyed,
 * and the free blocks of the devices' default memory pools.  A call never frees or
 * allocates scratch on the host's time: a cached buffer large enough is
 * reused with no allocator call; growth and eviction are stream-ordered
 * (hipFreeAsync / hipMallocAsync).  This trim is the one synchronising path:
 * it waits for each buffer's last use and for its device; a buffer a call is
 * using at that moment is kept.  No reference counterpart (the reference
 * allocates nothing).  Returns 0, or -3 with rdna_get_error() set. */
RDNA_API int32_t rdna_scratch_trim(void);

/* The scratch cache of HIP device `device`: bytes it holds, buffers it holds,
 * and the allocator calls (hipMallocAsync; hipMalloc for captured calls) the library
 * has made for that device's scratch since it was loaded.  For tests and monitoring;
 * no reference counterpart.  Returns 0, or -3 if an output pointer is null. */
RDNA_API int32_t rdna_scratch_stats(int32_t device, uint64_t* cached_bytes, int64_t* entries,
                                    int64_t* allocations);

/* Scratch of calls under stream capture is memory whose address is part of the graph:
 * each graph has its own, the calls captured on one stream share it, and it is handed on
 * to later captures, or freed by rdna_scratch_trim(), when the graph and its executables
 * are destroyed.  So two graphs may be replayed side by side, but not two copies
 * of one (executables instantiated from it, clones, child nodes), and a graph is
 * destroyed after its last replay has finished.  A larger call of the same capture
 * gets a block of its own, the smaller one stays for the graph's life.  The caps of
 * the cache do not count these blocks: this reads the bytes and the number of those
 * on `device`, owned or to be handed on.  Returns 0, or -3 if an output pointer is
 * null. */
RDNA_API int32_t rdna_graph_scratch_stats(int32_t device, uint64_t* bytes, int64_t* blocks);

/* rdna_attention_forward() for callers that cannot allocate device memory
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  No reference counterpart: the reference needs no scratch.
 * Same arguments, results and return codes as rdna_attention_forward(); the
 * scratch that path takes -- the RoPE-rotated K copy (B*Hkv*Sk*D fp16) and
 * the partials of split keys -- comes from a static 64 MiB device array the
 * library holds on each GPU it runs on, so the call makes no hipMalloc,
 * hipFree or pool allocation.  A call needing more than 64 MiB of scratch
 * returns -3 ("... bytes of scratch ...") before launching anything.  Every
 * call on one GPU shares that GPU's array: calls that overlap on a GPU
 * (different streams, not ordered) race. */
RDNA_API int32_t rdna_attention_forward_noalloc(
    const void* q, const void* k, const void* v, void* output,
    const void* rot_cos, const void* rot_sin,
    int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
    int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
    int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_s,
    int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s,
    uint32_t batch_size, uint32_t num_heads, uint32_t num_kv_heads,
    uint32_t seq_len, uint32_t key_seq_len, uint32_t head_dim,
    float scale, int32_t causal, int32_t has_rope, int32_t window_size,
    void* hip_stream);

/* Exact int32 scores S = Q_i8 K_i8^T (GQA head map kv = h / (Hq/Hkv)),
 * written to `scores`, a contiguous int32 [batch, num_heads, seq_len,
 * key_seq_len] device buffer.  Runs the INT8 attention kernel itself (its
 * score-export instantiation: the same K tile staging, LDS layout, operand
 * ring and v_mfma_i32_32x32x32_i8 sequence as rdna_attention_forward_int8qk's
 * first GEMM) and writes its accumulators; softmax, P V and output are
 * compiled out.  Key and query strides as for the forward (seq strides
 * <= 2^24 elements).  No reference counterpart: it exposes the production
 * kernel's scores so tests can check them bit for bit. */
RDNA_API int32_t rdna_int8_qk_scores(
    const void* q, const void* k, int32_t* scores,
    int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
    int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
    uint32_t batch_size, uint32_t num_heads, uint32_t num_kv_heads,
    uint32_t seq_len, uint32_t key_seq_len, uint32_t head_dim,
    void* hip_stream);

/* rdna_attention_forward_int8qk() with a per-channel V scale applied inside
 * the kernel: output = softmax-weighted sum of v_i8 * v_scale *
 * v_channel_vec[b, kv_head, d], where v_channel_vec is a contiguous fp32
 * [batch, num_kv_heads, head_dim] device array (16-byte aligned), or null for
 * the plain per-tensor v_scale.  No reference counterpart: the reference's
 * flash_attn_int8qk_quantized (rdnattention/__init__.py:346-357) multiplies
 * the kernel's fp16 output by v_channel in a separate torch pass; here that
 * product is part of the kernel's epilogue. */
RDNA_API int32_t rdna_attention_forward_int8qk_vchannel(
    const void* q, const void* k, const void* v, void* output,
    int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
    int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
    int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_s,
    int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s,
    uint32_t batch_size, uint32_t num_heads, uint32_t num_kv_heads,
    uint32_t seq_len, uint32_t key_seq_len, uint32_t head_dim,
    float scale, float q_scale, float k_scale, float v_scale,
    const void* q_scale_vec, const void* k_scale_vec, const void* v_channel_vec,
    int32_t causal, int32_t window_size, void* hip_stream);

/* rdna_attention_forward_int8qk() with a per-token V scale: V row j of each
 * (batch, kv head) is dequantised by v_token_vec[b, kv_head, j] while the
 * kernel stages it, v'_j = fp16(sat(v_i8[j] * v_token_vec[...])) (the product
 * in fp32, saturated to +-65504, rounded once to fp16), and the
 * quantised P (the reference's pq = min(127, round(127 p))) multiplies these
 * fp16 rows: output = sum_j pq_j v'_j * v_scale / (127 l).  v_token_vec is a
 * contiguous fp32 [batch, num_kv_heads, key_seq_len] device array (4-byte
 * aligned, required).  No reference counterpart: the reference lists a
 * per-token V scale as missing (FEATURES.md:191, :201-202); this is the extension
 * that fills it, with the per-token V quantiser of
 * quantize_int8_qk_pertoken's formula. */
RDNA_API int32_t rdna_attention_forward_int8qk_vtoken(
    const void* q, const void* k, const void* v, void* output,
    int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
    int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
    int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_s,
    int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s,
    uint32_t batch_size, uint32_t num_heads, uint32_t num_kv_heads,
    uint32_t seq_len, uint32_t key_seq_len, uint32_t head_dim,
    float scale, float q_scale, float k_scale, float v_scale,
    const void* q_scale_vec, const void* k_scale_vec, const void* v_token_vec,
    int32_t causal, int32_t window_size, void* hip_stream);

/* INT8 quantisation on the GPU, bit-identical to the reference wrapper's
 * torch ops (rdnattention/__init__.py:303-343):
 *   per_channel == 0 (per token): scale[b,h,s] = max_d |x| / 127 (0 -> 1)
 *   per_channel != 0 (per channel): scale[b,h,d] = max_s |x| / 127 (0 -> 1)
 *   q = clamp(round_half_even(x / scale), -127, 127)
 * x: fp16 (x_dtype 0) or fp32 (x_dtype 1) [batch, num_heads, seq_len,
 * head_dim] with element strides (b, h, s) and unit stride along head_dim;
 * 16-byte aligned, strides multiples of 16 bytes; head_dim a multiple of 8
 * up to 512.  q_out: int8 [batch, num_heads, seq_len, head_dim] contiguous;
 * scale_out: fp32, [batch, num_heads, seq_len] or [batch, num_heads,
 * head_dim], contiguous.
 * rot_cos / rot_sin (per token only; both or neither, nullptr = none): fp32
 * RoPE tables [>= seq_len, head_dim / 2], contiguous, 16-byte aligned, as
 * for rdna_attention_forward.  Each row (position s) is rotated first, with
 * the FP16 attention path's arithmetic (pairs rotated in fp32, rounded to
 * fp16 for fp16 input), and the rotated row is quantised: INT8 attention
 * with RoPE, which the reference does not offer.
 * Returns 0, or -3 with "Quantize (int8) failed: ...".
 * No reference counterpart (the reference quantises with torch ops). */
RDNA_API int32_t rdna_quantize_int8(
    const void* x, int32_t x_dtype,
    int64_t x_stride_b, int64_t x_stride_h, int64_t x_stride_s,
    uint32_t batch_size, uint32_t num_heads, uint32_t seq_len, uint32_t head_dim,
    int32_t per_channel, const void* rot_cos, const void* rot_sin,
    void* q_out, void* scale_out, void* hip_stream);

/* rdna_quantize_int8 of the Q, K and V of one attention call in one launch (two
 * with a per-channel V), the same values: q [batch, num_heads, seq_len,
 * head_dim] and k, v [batch, num_kv_heads, key_seq_len, head_dim], all of one
 * dtype; Q and K per token, rotated first when rot_cos / rot_sin are given, V
 * per channel (v_per_channel != 0) or per token.  Outputs and checks as for
 * rdna_quantize_int8.  No reference counterpart. */
RDNA_API int32_t rdna_quantize_int8_qkv(
    const void* q, const void* k, const void* v, int32_t dtype, int64_t q_stride_b, int64_t q_stride_h,
    int64_t q_stride_s, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s, int64_t v_stride_b,
    int64_t v_stride_h, int64_t v_stride_s, uint32_t batch_size, uint32_t num_heads, uint32_t num_kv_heads,
    uint32_t seq_len, uint32_t key_seq_len, uint32_t head_dim, int32_t v_per_channel, const void* rot_cos,
    const void* rot_sin, void* q_out, void* k_out, void* v_out, void* q_scale_out, void* k_scale_out,
    void* v_scale_out, void* hip_stream);

/* The kernels that a call of these sizes takes, for tests and measurements:
 * rdna_attention_forward (int8 == 0) or rdna_attention_forward_int8qk and its
 * variants (int8 != 0).  *form: 0 whole row tiles, 1 row tiles with their keys
 * split over workgroups, 2 the wave groups of a workgroup taking the key tiles
 * in turn, 3 split-K decode; *splits the key splits (0 where decode's cannot be
 * planned without a device), *scratch_bytes the bytes of their partials and,
 * for INT8, of the scores or row maxima.  max_partials limits the partials of
 * an FP16 call, as the rest of the no-allocation array does (UINT64_MAX: no
 * limit).  Launches nothing.  Returns 0, -3 (arguments) or -4 (built without
 * INT8).  No reference counterpart. */
RDNA_API int32_t rdna_attention_call_plan(
    int32_t int8, uint32_t batch_size, uint32_t num_heads, uint32_t num_kv_heads,
    uint32_t seq_len, uint32_t key_seq_len, uint32_t head_dim, int32_t causal, int32_t window_size,
    uint64_t max_partials, int32_t* form, int32_t* splits, uint64_t* scratch_bytes);

/* Kernel timer.  While enabled, each launch of a main attention kernel
 * (prefill, split-K, int8; not the RoPE pre-rotation or split-K combine
 * kernels) is bracketed by a HIP event pair recorded on its stream.
 * rdna_kernel_timer_enable(on) discards what was recorded and switches the
 * timer on (on != 0) or off.  rdna_kernel_timer_read waits for the recorded
 * events, stores the summed kernel time in *total_ms and the number of timed
 * launches in *launches, and clears the record; returns -3 if an event could
 * not be created, recorded or read.  Process-wide; no reference counterpart:
 * benchmarks use it to divide a kernel's FLOPs or bytes by its own time. */
RDNA_API int32_t rdna_kernel_timer_enable(int32_t on);
RDNA_API int32_t rdna_kernel_timer_read(double* total_ms, int64_t* launches);

/* ---------------------------------------------------------------------------
 * Paged key/value caches.  The reference has none.
 *
 * Keys and values live in pages of page_size tokens (a power of two): element
 * (page, token, head, channel) of the keys at key + page * key_stride[0] + token *
 * key_stride[1] + head * key_stride[2] + channel, strides in elements, multiples of
 * 16 bytes; the values likewise (append and commit refuse values at the keys' own
 * address).  Key j of sequence b is token j % page_size of page
 * block_tables[b * table_stride + j / page_size].  int8 pages have a float scale per
 * (page, token, head), strides in floats: the value is int8 * scale.
 *
 * seq_lens, block_tables and cu_seqlens are device memory that the host does not
 * read.  The newest rows of sequence b are the rows cu_seqlens[b] .. cu_seqlens[b +
 * 1] - 1 of a call's row tensors [num_rows, heads, head_dim] (cu_seqlens null:
 * num_rows / num_seqs each), n of them its keys seq_lens[b] - n .. seq_lens[b] - 1;
 * cu_seqlens begins with 0 and never falls (other values reach no row outside the
 * tensors, and give no defined result).
 * Rows behind the last sequence belong to none.  A length beyond the page table is
 * taken as the table's, a negative one as 0; the entry of a page that does not exist
 * never leads outside the pages (nothing is written for it, and what a call that
 * reads through it returns for that sequence is unspecified).
 * ------------------------------------------------------------------------- */
#define RDNA_DTYPE_F16 0
#define RDNA_DTYPE_BF16 1
#define RDNA_DTYPE_INT8 2
#define RDNA_DTYPE_F32 3 /* norm weights only */

typedef struct rdna_paged_cache {
    void* key;
    void* value;
    float* key_scale;   /* int8 pages only, else null */
    float* value_scale;
    const int32_t* block_tables; /* [num_seqs, table_width] */
    const int32_t* seq_lens;     /* [num_seqs], the newest rows among them */
    const int32_t* cu_seqlens;   /* [num_seqs + 1], or null */
    int64_t key_stride[3];       /* page, token, head */
    int64_t value_stride[3];
    int64_t key_scale_stride[3];
    int64_t value_scale_stride[3];
    int64_t table_stride;
    uint32_t num_pages, page_size, table_width, num_seqs, num_kv_heads, head_dim;
    int32_t dtype; /* RDNA_DTYPE_*; int8 at head_dim 64 and 128 */
} rdna_paged_cache;

/* Writes the newest rows' keys and values [num_rows, num_kv_heads, head_dim] (dtype:
 * fp16 or bf16; strides of rows and heads in elements) to their places in the pages;
 * int8 pages get the row quantised with its own scale (largest magnitude / 127, as
 * rdna_quantize_int8 does per token).  With rot_cos / rot_sin (float [rot_rows,
 * rot_dim / 2], 16-byte aligned) the first rot_dim channels of every key are rotated
 * first, by the angles of its index in the sequence or of positions[row]: channels
 * (2i, 2i + 1) by column i (rot_interleaved) or (i, i + rot_dim / 2); positions
 * outside the tables are taken as their first or last row.  With query, the query
 * rows [num_rows, num_heads, head_dim] are rotated likewise into query_out (query itself
 * with its strides, or memory that does not overlap it).  Rows without a place write
 * nothing; their query rows come out as they are (rotated if positions are given, and the
 * row is a sequence's).  rot_dim is a multiple of 16. */
RDNA_API int32_t rdna_paged_append(
    const rdna_paged_cache* cache, const void* key, const void* value, int64_t key_stride_row, int64_t key_stride_h,
    int64_t value_stride_row, int64_t value_stride_h, uint32_t num_rows, int32_t dtype, const void* query,
    void* query_out, int64_t query_stride_row, int64_t query_stride_h, int64_t query_out_stride_row,
    int64_t query_out_stride_h, uint32_t num_heads, const int32_t* positions, const void* rot_cos,
    const void* rot_sin, uint32_t rot_rows, uint32_t rot_dim, int32_t rot_interleaved, void* hip_stream);

/* What rdna_paged_append_norm does to queries and keys before they are rotated, and by
 * which positions. */
typedef struct rdna_paged_norm {
    const void* query_norm; /* [head_dim] weights, 16-byte aligned, or null */
    const void* key_norm;
    const int32_t* rot_axes;  /* [rot_dim / 2], or null: positions has one per row */
    int64_t position_stride;  /* with rot_axes: of the rows of positions [num_rows, num_axes] */
    uint32_t num_axes;
    float eps;
    int32_t dtype; /* RDNA_DTYPE_* of the weights: F32, or the rows' */
} rdna_paged_norm;

/* rdna_paged_append, where each head x of the queries (query_norm not null) and of the
 * keys (key_norm) first becomes x w / sqrt(mean(x^2) + eps), eps at least 0, and column c
 * of the tables turns by position rot_axes[c] of its row (outside 0 .. num_axes - 1: the
 * first or last), all in fp32 (of keys that are quantised in fp64) and rounded once.
 * query may be given without rot_cos and rot_sin where query_norm is.  Rows of no sequence
 * are not normed.  `norm` is read by the host. */
RDNA_API int32_t rdna_paged_append_norm(
    const rdna_paged_cache* cache, const rdna_paged_norm* norm, const void* key, const void* value,
    int64_t key_stride_row, int64_t key_stride_h, int64_t value_stride_row, int64_t value_stride_h, uint32_t num_rows,
    int32_t dtype, const void* query, void* query_out, int64_t query_stride_row, int64_t query_stride_h,
    int64_t query_out_stride_row, int64_t query_out_stride_h, uint32_t num_heads, const int32_t* positions,
    const void* rot_cos, const void* rot_sin, uint32_t rot_rows, uint32_t rot_dim, int32_t rot_interleaved,
    void* hip_stream);

/* softmax(scale Q K^T) V of the newest rows over the pages, head_dim a multiple of 32
 * up to 256, query and output fp16 or bf16 (dtype; the pages' own type, or any with
 * int8 pages).  causal and window_size as in rdna_attention_forward.  A row that sees
 * no key is zeros.  max_rows_per_seq: most rows of a sequence as far as the caller
 * knows (num_rows if not); it picks kernels, which round in other places, and decides
 * nothing else.  Calls that could have 2^31 key tiles are refused, before anything is
 * launched: about rows x num_heads x keys of the table beyond 2^45 (2^44 above head_dim
 * 128), or num_seqs x num_kv_heads x keys of the table beyond 2^36.
 *
 * With tree_mask ([num_seqs, tree_n, tree_n] bytes, 0 or 1, strides of sequences and
 * rows in bytes) the newest rows are drafts: row i sees every key before the drafts
 * and draft j where tree_mask[b][i][j]; causal and window_size must be off.
 *
 * The rows of output behind the last sequence are left as they are, or set to zeros
 * (zero_tail).  The scratch is stream-ordered like the split-K partials'. */
RDNA_API int32_t rdna_paged_attention(
    const rdna_paged_cache* cache, const void* query, void* output, int64_t query_stride_row, int64_t query_stride_h,
    int64_t output_stride_row, int64_t output_stride_h, uint32_t num_rows, uint32_t num_heads, int32_t dtype,
    uint32_t max_rows_per_seq, float scale, int32_t causal, int32_t window_size, const uint8_t* tree_mask,
    int64_t tree_stride_seq, int64_t tree_stride_row, uint32_t tree_n, int32_t zero_tail, void* hip_stream);

/* Prefixes that sequences share, in the pages of the same cache: the first lens[i] keys
 * of table row i come before the own keys of sequences seqs[i] .. seqs[i + 1] - 1 (seqs
 * [num_prefixes + 1], from 0 to the number of sequences and never falling; null: one
 * prefix, of all of them).  All of it device memory that the host does not read; a
 * length of 0 is no prefix. */
typedef struct rdna_paged_prefix {
    const int32_t* block_tables; /* [num_prefixes, table_width] */
    const int32_t* lens;         /* [num_prefixes] */
    const int32_t* seqs;
    int64_t table_stride;
    uint32_t table_width, num_prefixes;
} rdna_paged_prefix;

/* rdna_paged_attention of rows that see their sequence's prefix too (prefix not null):
 * all of it, whatever causal hides of the sequence's own keys; without window_size.  A
 * prefix is read once for all of its sequences.  lse, if not null: float [num_rows,
 * num_heads], the logarithm of the sum of exp(score) over the keys that a row sees, -inf
 * where there is none; of the rows behind the last sequence (where cu_seqlens is given)
 * -inf whether or not zero_tail is set.  The prefixes' part of every row is scratch: num_rows
 * x num_heads x (head_dim + 1) floats (of calls with few rows up to 18 MB), above 256 MiB
 * allocated anew by every call (hipMallocAsync); without that memory the call fails with
 * -3, before it has written anything. */
RDNA_API int32_t rdna_paged_attention_lse(
    const rdna_paged_cache* cache, const rdna_paged_prefix* prefix, const void* query, void* output,
    int64_t query_stride_row, int64_t query_stride_h, int64_t output_stride_row, int64_t output_stride_h,
    uint32_t num_rows, uint32_t num_heads, int32_t dtype, uint32_t max_rows_per_seq, float scale, int32_t causal,
    int32_t window_size, int32_t zero_tail, float* lse, void* hip_stream);

/* Keeps accepted drafts: for every sequence, key and value prefix_lens[b] + i become
 * those of prefix_lens[b] + path[b * path_stride + i], i < path_lens[b] (at most
 * path_n <= 1024), all of them read before the first is written; entries below 0
 * and keys beyond the table move nothing.  cache->seq_lens and cu_seqlens are not
 * looked at.  At most 65535 sequences. */
RDNA_API int32_t rdna_paged_commit(const rdna_paged_cache* cache, const int32_t* prefix_lens, const int32_t* path,
                                   int64_t path_stride, uint32_t path_n, const int32_t* path_lens,
                                   void* hip_stream);

/* Adds the attention that each key has received from the newest rows to its weight:
 *   w = (decay w, or 0 where the key is one of the newest rows' own)
 *       + sum over the rows and the heads of the key's kv head of exp(score - lse)
 * with lse [num_rows, num_heads] as rdna_paged_attention_lse gives it (a row of -inf adds
 * nothing) and scores, causal and window_size as there; over the cache's own keys alone
 * where the rows saw a prefix too.  key_weights: float (page, token, head) with
 * key_weights_stride in floats, none of them 0 where there are several.  decay at least 0; with 0
 * the old weights are not read.  Sequences without rows, and places without a key, are left
 * as they are.  No page may belong to two sequences with rows: the sums of one of them could
 * be lost.  The values of the cache are not looked at.  The same bits every time. */
RDNA_API int32_t rdna_paged_key_weights(
    const rdna_paged_cache* cache, const void* query, int64_t query_stride_row, int64_t query_stride_h,
    uint32_t num_rows, uint32_t num_heads, int32_t dtype, uint32_t max_rows_per_seq, const float* lse, float scale,
    int32_t causal, int32_t window_size, float decay, float* key_weights, const int64_t* key_weights_stride,
    void* hip_stream);

/* Keeps `budget` keys of every sequence that has more, for each kv head its own: the
 * `first` first ones, the `recent` newest ones and, of those between, the ones of the
 * largest weights (of equal ones those in front; a weight that is not a number is below
 * all).  In their order they move up to the front of the sequence, with their values,
 * scales and weights; what is behind them then is unspecified.  new_lens [num_seqs]
 * (not seq_lens itself): the lengths after it, min(length, budget); kept [num_seqs,
 * num_kv_heads, budget]: which keys they were, -1 behind the last.  No page may belong to
 * two sequences.  Where a table names a page that does not exist, the weight counts as
 * below all and nothing moves.  At most 65535 sequences. */
RDNA_API int32_t rdna_paged_evict(const rdna_paged_cache* cache, float* key_weights,
                                  const int64_t* key_weights_stride, uint32_t budget, uint32_t first, uint32_t recent,
                                  int32_t* new_lens, int32_t* kept, void* hip_stream);

/* Library version string ("0.1.0-gfx950"). */
RDNA_API const char* rdna_version(void);

#endif /* RDNATTENTION_EXT_H */
