/*
 * needle_engine.h — the model-level C ABI under needle.h: the contract the
 * reference's engine crate gives its agent, CLI and benches (Model, Session,
 * head logits), made batched so one call advances many independent
 * sequences on one GPU. Plain pointers and sizes only.
 *
 * Each entry names the reference interface it replaces (file:line in
 * needle-rs). A batch holds S sequences that are fed in lockstep: every call
 * gives each sequence the same number of new tokens, so they share positions.
 * A batch is driven by one host thread at a time.
 *
 * Pointers: with ND_DEVICE in `flags` the id/mask/output pointers are device
 * pointers on the model's GPU and the call is asynchronous on the batch's
 * stream; otherwise they are host pointers, copied in and out inside the
 * call, which returns when the results are in host memory.
 */
#ifndef NEEDLE_ENGINE_H
#define NEEDLE_ENGINE_H

#ifdef __cplusplus
extern "C" {
#endif

typedef struct nd_model nd_model;
typedef struct nd_batch nd_batch;

enum { ND_DEVICE = 1 };

/* crates/needle-engine/src/model.rs:150-160 (`Outputs`). */
enum {
    ND_OUT_NONE = 0,        /* Outputs::None */
    ND_OUT_LAST_LOGITS = 1, /* Outputs::LastLogits: [S][out_rows] */
    ND_OUT_LAST_HIDDEN = 2, /* Outputs::LastHidden: [S][d_model] */
    ND_OUT_ALL_LOGITS = 3,  /* Outputs::AllLogits: [S][t][out_rows] */
    ND_OUT_HIDDEN = 4       /* Outputs::Hidden: [S][t][d_model] */
};

/* crates/needle-engine/src/loader.rs:40-59 with weights.rs:314-497
 * (Weights::from_archive_mode, fast) and model.rs:248-253 (Model::quantized):
 * parse the archive, upload its packed matrices and small weights to GPU
 * `device`, build the int8 gate projection and RoPE tables. The archive
 * bytes are only read during the call. 0 on success, -1 on error. */
int nd_model_load(const unsigned char* cact, unsigned long long n, int device, nd_model** out);
void nd_model_free(nd_model* m);

/* crates/needle-core/src/cact.rs:173-202 (Header::to_config): dims[0..9] =
 * vocab, out_rows, d_model, num_layers, num_heads, num_kv_heads,
 * qk_head_dim, v_head_dim, max_seq_len. */
int nd_model_dims(const nd_model* m, int* dims);

/* model.rs:264-274 (Model::session), for `num_seqs` sequences of up to
 * `max_len` positions each. `max_len` must lie in [1, max_seq_len] and be
 * at most 8192 (the attention kernel holds 32 key chunks of 256); beyond
 * that the call fails with a message, as a too-long session does. */
int nd_batch_new(nd_model* m, int num_seqs, int max_len, nd_batch** out);
void nd_batch_free(nd_batch* b);

/* model.rs:72-74 (Session::len): positions every sequence has been fed. */
int nd_batch_len(const nd_batch* b);

/* Session::attend (crates/needle-engine/src/model.rs:63-66, infer.rs:
 * 1749-1825) for every sequence of the batch: each query sees the first
 * `sink` positions within its layer's band, then the positions from
 * max(chunk end - ring, sink) on (the engine's ring, which the band does
 * not cut), as the agent sets it (agent.rs:583-588: sink = the static
 * prefix, ring = the header's kv_window). ring = 0 restores plain
 * attention. Rollbacks are not served, so every position in those runs
 * still holds its keys (the batch's cache keeps all max_len positions). */
int nd_batch_set_attend(nd_batch* b, int sink, int ring);

/* Session::rollback (model.rs:81-113, infer.rs:1055-1077): drop the last
 * n <= 32 positions of every sequence without recomputing; the next feed
 * continues from there (conv and engram histories, RoPE rows and KV of the
 * kept positions stay). Fails, changing nothing, when under the batch's
 * attention span a kept position's ring slot holds a dropped position (the
 * reference would skip that key and re-feed it, which is not served). */
int nd_batch_rollback(nd_batch* b, int n);

/* Session::rewind_zeroed (model.rs:116-126, infer.rs:1039-1053): forget
 * positions len.. as the engine's context-overflow re-feed does: the KV
 * cache keeps what it holds, the conv history and RoPE rows start over.
 * The same refusal as nd_batch_rollback. */
int nd_batch_rewind_zeroed(nd_batch* b, int len);

/* Session::truncate (model.rs:128-145): drop everything past len; up to 32
 * positions by nd_batch_rollback, more by feeding the first len tokens to
 * fresh sessions again (which, as in the reference, have no attention
 * span). */
int nd_batch_truncate(nd_batch* b, int len);

/* model.rs:304-306 (Model::forward) through infer.rs:1105-1131
 * (forward_native): feed ids[S][t] to every sequence in the engine's chunks
 * of at most 32, writing `outputs` to out (may be NULL for ND_OUT_NONE).
 * Returns the rows written per sequence, -1 on error. */
int nd_batch_forward(nd_batch* b, const int* ids, int t, int outputs, float* out, int flags);

/* The greedy decode loop of crates/needle-cli/src/main.rs:577-581 and
 * generate.rs:110-125, with the agent's ban (agent.rs:1114-1127): for each
 * sequence take the first index of the maximum of its last logits after the
 * ids its mask disallows read -1e30 (allow_bits [S][ceil(out_rows/8)], bit
 * set = allowed, LSB first; NULL allows all), write it to next_ids[S], and
 * feed it as one decode step. Needs a preceding forward with logits. */
int nd_batch_step(nd_batch* b, const unsigned char* allow_bits, int* next_ids, int flags);

/* infer.rs:1016 (NatState::last_hidden): each sequence's final normed hidden
 * state of the last position a forward returned outputs for, [S][d_model]. */
int nd_batch_last_hidden(nd_batch* b, float* out, int flags);

/* infer.rs:1135-1141 (Model::head_logits): logits of h[rows][d_model] with
 * the decode kernel, out[rows][out_rows]. */
int nd_head_logits(nd_batch* b, const float* h, int rows, float* out, int flags);

/* infer.rs:1145-1166 (Model::head_logits_sparse): one row h[d_model]; the
 * ids are scored with the single-row kernel, every other entry is NEG
 * (0xf149f2ca). out[out_rows]. Host pointers. */
int nd_head_logits_sparse(nd_batch* b, const float* h, const int* ids, int n, float* out);

/* The start of the agent's grammar-constrained call step, per sequence,
 * over logits[S][out_rows] (NULL = the batch's last logits; the agent's
 * sparse-logit rows, agent.rs:390-420, come in this way)
 * (crates/needle-engine/src/agent.rs:295-343):
 * entries whose bit in `allow` is clear read -1e30 (the step's bans; NULL =
 * none), and over that m[s] = the max and z[s] = sum exp(l - m) as
 * softmax_stats forms them (agent.rs:1241-1252: four f32 lanes of the
 * engine's exp over whole groups of four, then the remainder in f64).
 * Entries whose bit in `allow_order` is also clear (the call step's further
 * bans; NULL = none) leave the candidates: live[s] = how many logits
 * exceed -1e30 and ids[s][0..k) the first k of them by logit, lowest id
 * first on ties (the top-128 partial selection and sort, agent.rs:335-343),
 * -1 past live. 1 <= k <= 128; masks [S][ceil(out_rows/8)], bit set =
 * allowed. The grammar's accept test that walks these candidates stays on
 * the host. Host pointers, or device pointers with ND_DEVICE. */
int nd_batch_candidates(nd_batch* b, const float* logits, const unsigned char* allow, const unsigned char* allow_order,
                        int k, int* ids, float* m, double* z, int* live, int flags);

/* needle_embed's computation after tokenizing (crates/needle-engine/src/
 * heads.rs:63-90, agent.rs:259-263) for every sequence of a fresh batch
 * (nothing fed yet): ids[S][T] are fed in chunks of 32 recording the lane
 * mean of the residual stream at every position and depth (the cells,
 * infer.rs:1195-1211), then the probe pool of the embedding head,
 * projected and scaled to unit norm (without an embedding head, the
 * confidence head's pool at unit norm). out[S][dim]; with out == NULL only
 * *dim is set. Fails without a probe head ("this archive carries no probe
 * head"). The batch keeps the T fed positions. Host or device pointers
 * (ND_DEVICE). */
int nd_batch_embed(nd_batch* b, const int* ids, int T, float* out, int* dim, int flags);

/* heads.rs:68-74 (confidence_logit) the same way: out[S] = the confidence
 * head's logit for each sequence of a fresh batch. */
int nd_batch_confidence(nd_batch* b, const int* ids, int T, float* out, int flags);

/* The CUDA stream a batch's work runs on (a cudaStream_t); no counterpart
 * in the reference, which runs on the CPU. */
void* nd_batch_stream(nd_batch* b);

/* crates/needle-core/src/quant.rs:233-256 (cq_pack, group 128) at bits 2,
 * 3, 4 or 5 (ternary; quant.rs:11-12): w[rows][d] to codes[rows][G * 16 *
 * width] (G = ceil(d/128), width = bits, 2 for ternary; LSB-first) and f16
 * norms[rows][G]. The reference's packer takes bits 4 only; the other widths
 * are written in the layout its loader reads (qlinear.rs:220-236). */
int nd_cq_pack(const float* w, int rows, int d, int bits, unsigned char* codes, unsigned short* norms);

/* Test and benchmark support: one CQ matrix (codes [out][6][16 * width],
 * f16 norms [out][6] as nd_cq_pack writes them at `bits`; in_dim 768) on GPU
 * `device`, and the engine's matmul of host rows x[M][768] into y[M][out]:
 * each row quantized as QAct::new (qlinear.rs:152-207), then the decode
 * combine (qlinear.rs:340-350) when T == 1, else the prefill combine
 * (qlinear.rs:353-363) over consecutive sequences of T rows (M a multiple
 * of T). With reps > 0 and ms != NULL it also times reps back-to-back runs
 * (A8 + matmul, inputs resident) and stores the mean in *ms. */
typedef struct nd_cqmat nd_cqmat;
int nd_cqmat_new(int device, const unsigned char* codes, const unsigned short* norms, int out, int in_dim, int bits,
                 nd_cqmat** out_mat);
void nd_cqmat_free(nd_cqmat* mat);
int nd_cqmat_apply(nd_cqmat* mat, const float* x, int M, int T, float* y, int reps, float* ms);
/* Benchmark support: the matmul alone (no A8), launched back to back over
 * the n matrices in turn, `reps` rounds after one untimed round, on the
 * activations the last nd_cqmat_apply of mats[0] quantized (M <= its rows).
 * When the matrices together exceed L2 every launch streams its weights
 * from HBM. *ms = mean time per launch. The matrices share device and
 * shape. */
int nd_cqmat_time_rotating(nd_cqmat* const* mats, int n, int M, int T, int reps, float* ms);

/* crates/needle-core/src/cact.rs:399-475 (pack) over random-init Needle 3
 * weights: every tensor ~N(0, std^2), seeded; CQ matrices, f16 small
 * weights, MT19937 Hadamard permutations. Shape knobs let tests shrink the
 * model (num_layers, vocab, engram_slots, sliding_window; engram_sites is
 * a bit mask of layers, global_mask likewise). cq_bits[i] is the record
 * bits (2, 3, 4, 5 = ternary) of the i-th CQ record in record order, 4 past
 * n_cq_bits (a mixed-width archive; the reference's packer writes one
 * width). heads_mask bit c appends probe head c (1 embedding, 2
 * confidence, 3 router; cact.rs:354-392: 4 probes a depth, 4 queries, the
 * embedding head 128 wide). With out == NULL returns the byte size in
 * *len; else writes up to cap bytes. */
int nd_synth_cact(int num_layers, int vocab, int engram_slots, int sliding_window, unsigned long long global_mask,
                  unsigned long long engram_sites, unsigned long long seed, float std, const int* cq_bits, int n_cq_bits,
                  unsigned heads_mask, unsigned char* out, unsigned long long cap, unsigned long long* len);

/* Kernel launches this process has issued (all batches, all devices); no
 * counterpart in the reference. */
long long nd_launch_count(void);

/* Launch sites whose kernels can be timed with CUDA events on the batch's
 * stream (no counterpart in the reference): nd_batch_time_site(b, site)
 * starts recording every launch of that site (clearing earlier records;
 * ND_SITE_NONE stops), nd_batch_site_time() waits for the stream and
 * returns the summed kernel time and the number of launches. Two sites share
 * launches in small batches: with at most one row an SM, each layer's post
 * block launch also runs the next layer's mHC read (ND_SITE_POST covers
 * both; ND_SITE_MHC times layer 0's alone), and one-token steps of up to
 * four sequences run the q|k|v|gate projection with the conv (ND_SITE_QKVG
 * covers both; ND_SITE_CONV records none). */
enum {
    ND_SITE_NONE = 0,
    ND_SITE_QKVG = 1,      /* q|k|v|gate projection */
    ND_SITE_OUT = 2,       /* attention out projection */
    ND_SITE_LM_HEAD = 3,   /* tied lm_head logits */
    ND_SITE_ENGRAM_KV = 4, /* engram key|value projection */
    ND_SITE_ATTENTION = 5, /* int8 KV attention + gate */
    ND_SITE_POST = 6,      /* post block: norms, Hadamard MLP, Sinkhorn, mHC write */
    ND_SITE_MHC = 7,       /* mHC read, engram gate, input norm, A8 */
    ND_SITE_CONV = 8       /* conv taps, head norm, RoPE, int8 KV write */
};
int nd_batch_time_site(nd_batch* b, int site);
int nd_batch_site_time(nd_batch* b, double* total_ms, int* launches);

/* No counterpart in the reference. nd_head_logits without any allocation,
 * for callers that cannot call cudaMalloc (their GPU memory belongs to
 * another allocator, or they must not take cudaMalloc's implicit device
 * synchronisation): logits of h[rows][d_model] into out[rows][out_rows] with
 * the decode kernel, both device pointers on the model's GPU, queued on
 * `stream` (a cudaStream_t; NULL is the legacy default stream) and not
 * waited for. The int8 activations live in one static device array of the
 * library, so rows is limited to 1..64; larger requests return -1 with the
 * reason in nd_last_error(). The first call on each device looks up that
 * array's device address, so make it before capturing any stream into a
 * CUDA graph. All calls share the array: calls whose work overlaps on the
 * GPU (other streams, other threads) race; the array keeps the last call's
 * contents, none of which the next call reads before writing. */
int nd_head_logits_noalloc(const nd_model* m, const float* h, int rows, float* out, void* stream);

/* The fused row ops of a layer as standalone kernels (BASELINE's fused-ops
 * sweep; in the forward pass they are fused into larger kernels). Device
 * pointers, queued on `stream` (a cudaStream_t; NULL = the legacy default
 * stream) and not waited for; 0 on success, -1 with nd_last_error().
 * Float pointers must be 16-byte aligned. */

/* infer.rs:426-443 (zcn, the zero-centred RMSNorm) with infer.rs:372-417
 * (dot16): out[t] = fma(x[t] r, s, x[t] r), r = 1 / sqrt(dot16(x[t],
 * x[t]) / 768 + 1e-6), for rows x[T][768] and weights s[768]. */
int nd_op_zcn(const float* x, const float* s, int T, float* out, void* stream);

/* The rotary embedding of a chunk's rows (infer.rs:1474-1483 with the
 * tables of infer.rs:938-946 and 1716-1744) at positions 0 .. T-1: x[T][672]
 * holds 12 query heads then 2 key heads of 48; in each, x[f] and x[f + 24]
 * (f < 24) rotate by the angle freq[f] * t, freq[f] = powf(theta,
 * f * (-2 / 48)). out may equal x. */
int nd_op_rope(const float* x, int T, float theta, float* out, void* stream);

/* infer.rs:2463-2496 (silu_native): out[i] = x[i] / (nexp(-x[i]) + 1) for
 * n elements (the Hadamard MLP's activation). */
int nd_op_silu(const float* x, long long n, float* out, void* stream);

/* qlinear.rs:309-323 (QMat::row) of the model's token embedding for each of
 * ids[T] (device int32): out[T][d_model], the codes dequantized by their
 * f16 group norms and rotated back (without the forward's sqrt(d_model)
 * scale). An id outside [0, vocab) gives a row of zeros. */
int nd_op_gather(const nd_model* m, const int* ids, int T, float* out, void* stream);

/* ---- Serving from one pool of pages: a 4-bit cache shared by sequences of
 * different lengths, attention over it, page bookkeeping, draft checking.
 * No counterpart in the reference, whose cache is one session's int8 ring.
 * Device pointers of GPU `device`, whichever device is current; queued on
 * `stream` (of that device; NULL = its legacy default stream) and not waited
 * for; 0 on success, -1 with nd_last_error() and nothing that would write a result queued. No call
 * allocates or keeps anything, so all may be captured into a graph; a
 * workspace `ws` is the caller's, holds nothing between calls, and must not
 * be used by two calls that overlap on the GPU. Lengths, tables and ids are
 * read on the device and may change between replays; whatever they hold, no
 * kernel reads or writes outside the buffers named here. */

/* Types of rows and logits. */
enum { ND_F32 = 0, ND_F16 = 1, ND_BF16 = 2 };
/* In `flags`: output rows behind the last sequence are set to zero instead
 * of left as they were. */
enum { ND_ZERO_REST = 2 };

/* A 4-bit cache and the rows of one call. pool: num_pages pages,
 * page_stride bytes apart (a multiple of 16; the pointer 16-byte aligned),
 * each [heads][page / 16] tiles of 16 * (dk / 2 + dv / 2 + 8) bytes: key codes
 * [16][dk / 2], value codes [16][dv / 2] (two a byte, lower dimension in the
 * low nibble), f16 (scale, minimum) of the 16 keys, of the 16 values; a value
 * is minimum + scale * code. page is a multiple of 16; (dk, dv) is (48, 64),
 * (64, 64) or (128, 128); at most 2^20 sequences. table[seqs][max_pages]
 * (rows table_stride apart) names each sequence's pages in order; positions
 * past its columns, or on a page id outside [0, num_pages), do not exist.
 * lens[seqs]: positions each sequence holds, this call's rows included. The
 * call's `rows` rows belong to the sequences in order, start[s] .. start[s +
 * 1] - 1 to sequence s (start[seqs + 1], ascending from 0; NULL: rows / seqs
 * each): row i of the n of sequence s is position lens[s] - n + i. Rows behind
 * start[seqs] are left
 * alone. */
typedef struct nd_kv4 {
    int device;
    void* pool;
    long long page_stride;
    int num_pages, page, heads, dk, dv;
    const int* table;
    int table_stride, max_pages, seqs;
    const int* lens;
    const int* start;
    int rows;
} nd_kv4;

/* Quantize rows k[rows][heads][dk], v[rows][heads][dv] of `type` (element
 * strides k_row, k_head, ..; the last dimension contiguous) into their
 * places. Per row and head, in f32: scale = f16(min((max - min) / 15, 65504)),
 * minimum = f16(min, clamped to +-65504), code = rint((x - minimum) / scale)
 * in [0, 15], 0 where scale is 0. A row of values holding a NaN or an infinity
 * is stored as NaN. Rows whose position does not exist are dropped. Two rows
 * of one call given the same place (a page that two sequences share: fork it
 * first) leave a mixture. */
int nd_op_kv4_append(const nd_kv4* kv, int type, const void* k, long long k_row, long long k_head, const void* v,
                     long long v_row, long long v_head, void* stream);

/* The cache's values at the rows' positions, rounded once to `type`; zeros
 * where a position does not exist. */
int nd_op_kv4_read(const nd_kv4* kv, int type, void* k, long long k_row, long long k_head, void* v, long long v_row,
                   long long v_head, int flags, void* stream);

/* Attention of the rows q[rows][q_heads][dk] over the cache (which holds the
 * rows' own keys already): out[rows][q_heads][dv] of the same `type`. Query
 * head g reads kv head g / (q_heads / heads), q_heads / heads <= 64. A row at
 * position p sees the positions j <= p that exist, with window > 0 only those
 * with j > p - window or j < sink. out = softmax(scale q.k) v; zeros for a row
 * that sees nothing. Scores are held in f32: queries beyond 2^100 may give NaN.
 * out must not overlap q. ws:
 * nd_op_kv4_attend_ws(the same arguments) bytes, 16-byte aligned; NULL where
 * that is 0. */
unsigned long long nd_op_kv4_attend_ws(const nd_kv4* kv, int type, int q_heads, int window, int sink);
int nd_op_kv4_attend(const nd_kv4* kv, int type, const void* q, long long q_row, long long q_head, int q_heads, float scale,
                     int window, int sink, void* out, long long o_row, long long o_head, void* ws, unsigned long long ws_bytes,
                     int flags, void* stream);
/* The waits inside the kernel for prompts of 16-bit rows are bounded. Should
 * one run out, which takes a fault elsewhere, what is left of its block's rows
 * is NaN and the call still returns 0. This sets the bound, in rounds, for the
 * calls of this process from here on and returns what it was: for tests. */
unsigned nd_op_kv4_attend_wait_rounds(unsigned rounds);

/* A pool as bytes: page p of layer l lies at pool + p * page_stride + l *
 * layer_stride, page_bytes long (all multiples of 16; pool 16-byte aligned;
 * pages do not overlap; at most 2^28). A nd_kv4 pool is one layer of it. */
typedef struct nd_pages {
    int device;
    void* pool;
    long long page_stride, layer_stride, page_bytes;
    int num_pages, layers;
} nd_pages;

/* From a table of old sequences to one of new ones: forking, truncating,
 * growing and freeing in one call. New sequence d (of n) keeps the first
 * keep[d] positions of old sequence src[d] (none where src[d] is not in
 * [0, seqs)) and gets room for need[d]; both are cut to the row's cols * page
 * positions, need to keep at least. Whole kept pages are shared. A kept page
 * that is partly filled and will be written (need > keep) is copied, in
 * every layer, unless d alone refers to it, or all that refer to it will
 * write on it and d is the first of them. Pages that no new sequence refers
 * to and whose pinned[] byte (num_pages, may be NULL) is 0 are free; fresh
 * pages are the free ones in ascending order, given to the new sequences in
 * order, each first its copy, then its columns. Pinned pages are never
 * written: they count as referred to by one more that does not write.
 * table_out[n][cols] (not the old table): -1 where there is no page, where a
 * kept entry was outside [0, num_pages), and where free pages ran out.
 * refs[num_pages]: references from table_out. info[4]: pages referred to or
 * pinned, fresh pages given, copies made, fresh pages wanted but not had.
 * The call reads the old table only, and overwrites free pages alone, so it
 * may be repeated. ws: nd_op_pages_fork_ws bytes, 16-byte aligned. */
unsigned long long nd_op_pages_fork_ws(int num_pages, int n);
int nd_op_pages_fork(const nd_pages* pool, const int* table, int table_stride, int seqs, int cols, int page, const int* src,
                     const int* keep, const int* need, int n, const unsigned char* pinned, int* table_out, int* refs, int* info,
                     void* ws, unsigned long long ws_bytes, void* stream);

/* Live pages (in the table, or pinned) to the front: with n of them, those
 * at ids >= n that are not pinned move, in ascending order, to the ids < n
 * that are not live. table_out[seqs][cols] (not the old table): the new
 * ids, -1 for entries outside [0, num_pages). map[num_pages]: each live
 * page's new id, -1 for the others. info[2]: n, pages moved. Moved pages'
 * old places keep their bytes. ws as above. */
unsigned long long nd_op_pages_compact_ws(int num_pages);
int nd_op_pages_compact(const nd_pages* pool, const int* table, int table_stride, int seqs, int cols, const unsigned char* pinned,
                        int* table_out, int* map, int* info, void* ws, unsigned long long ws_bytes, void* stream);

/* Check drafted tokens against the target and draw the next one, for each
 * of seqs sequences. logits (of `type`; element strides l_seq, l_row): row i
 * of T + 1 is the target's for the place of draft[s][i], row counts[s] for
 * the token after the last one. counts[seqs] (NULL: T each; cut to [0, T])
 * says how many of draft[seqs][T] there are; T <= 64. p_i = softmax(logits_i /
 * temperature[s]), or one at the first largest logit where the temperature
 * is not above 0 (+infinity: all logits above -infinity alike). q[seqs][T][V] f32 (strides q_seq, q_row; NULL: the draft
 * was certain of its tokens): the draft's probabilities. u[seqs][T + 1] in
 * [0, 1). Draft i is accepted, while all before it are, if u[i] q_i(draft_i)
 * < p_i(draft_i). The next token is drawn from max(p_i - q_i, 0) (p_i if that
 * is all zero) at the first i refused, from p after the last: the first j
 * whose running sum over 0 .. j exceeds u[T] times the whole. accepted[seqs];
 * tokens[seqs][T + 1]: the accepted drafts, the drawn token, then -1;
 * probs[seqs][T + 1]: p of each of them (the drawn one's rounded once, an
 * accepted draft's within 1e-5 of itself), then 0. A row that holds a NaN, a
 * +infinity at a temperature above 0, or nothing above -infinity accepts
 * nothing and draws -1 with probability 0; so does a residual that holds a
 * NaN. A drafted id outside [0, V) is refused. Sums and comparisons that
 * decide are exact to f64 rounding. At most 2^20 sequences,
 * V at most 2^30. ws: nd_op_verify_ws(seqs, T, V) bytes, 16-byte aligned. */
unsigned long long nd_op_verify_ws(int seqs, int T, int V);
int nd_op_verify(int device, int type, const void* logits, long long l_seq, long long l_row, const int* draft,
                 const int* counts, const float* u, const float* temperature, const float* q, long long q_seq,
                 long long q_row, int seqs, int T, int V, int* tokens, int* accepted, float* probs, void* ws, unsigned long long ws_bytes,
                 void* stream);

/* The last failure on this thread (empty if none). */
const char* nd_last_error(void);

/* Test support: copy an internal per-row buffer of the last forward
 * ("xs", "u", "p", "x1", "proj", "qbuf", "att", "o", "h", "logits", or the
 * same names snapped after layer `layer` when nd_batch_debug_layer(b, layer)
 * was set, prefixed "snap."). Returns the float count, -1 if unknown. */
int nd_batch_debug(nd_batch* b, const char* name, float* out, long long cap);
int nd_batch_debug_layer(nd_batch* b, int layer);

#ifdef __cplusplus
}
#endif

#endif /* NEEDLE_ENGINE_H */
