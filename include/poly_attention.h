/*
 * poly_attention.h -- C ABI of libpolyattn.so, the B200 (sm_100a) poly-attention
 * hot path.
 *
 * Every entry point is stream-ordered (it only enqueues work on `stream`, a
 * cudaStream_t passed as void*), allocates no device memory, keeps no
 * per-call state, and returns one of the POLY_* status codes below. On a
 * non-zero status, poly_last_error() returns a message for the calling thread.
 *
 * Layout convention for every tensor argument: element strides are given for
 * the (batch, head, row) axes; the last (feature) axis is contiguous. Score
 * rows are queries i, columns are keys j. Grouped-query attention: query head
 * h reads key/value head h / (heads / kv_heads).
 *
 * Reference interfaces replaced (lucidrains/poly-attention 0.3.6):
 *   poly_pass_fwd  <- _poly_flash_fwd_kernel launch
 *                     (poly_attention/flash_poly_attention.py:21-154, launched
 *                     at :347-359 for pass 1 and :365-377 for pass 2), and the
 *                     materialised passes of reference_poly_attention
 *                     (poly_attention/poly_attention.py:63-114) incl. masks
 *   poly_pass_bwd  <- _poly_flash_bwd_kernel launch
 *                     (poly_attention/flash_poly_attention.py:164-316, launched
 *                     at :409-422 and :429-442) plus the dq2 sum at :444
 *   poly_lse_merge <- no counterpart: merges key-split partial passes (the
 *                     long-context sequence split across GPUs)
 *   poly_decode_chain <- the cached passes of one decoding step, run level
 *                     after level (poly_attention/n_poly_attention.py:263-313,
 *                     poly_attention/poly_attention.py:63-114 with cache)
 */
#ifndef POLY_ATTENTION_H_
#define POLY_ATTENTION_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define POLY_ABI_VERSION 2

#if defined(__GNUC__)
#define POLY_API __attribute__((visibility("default")))
#else
#define POLY_API
#endif

/* status codes */
#define POLY_OK 0
#define POLY_EINVAL 1        /* bad shape, stride, dtype or pointer */
#define POLY_EUNSUPPORTED 2  /* valid request this build has no kernel for */
#define POLY_ECUDA 3         /* a CUDA call failed (launch, attribute, driver) */

/* element types */
#define POLY_F32 0
#define POLY_F16 1
#define POLY_BF16 2

/*
 * One attention pass with an additive per-key bias, emitting per-row
 * log-sum-exp. Both passes of order-2 poly attention and every level of the
 * order-n chain are instances of it:
 *
 *   s_ij  = scale * q_i . k_j ; if softclamp > 0: s_ij = c * tanh(s_ij / c)
 *   masked (causal j > i, key_mask[j] == 0, query_mask[i] == 0) -> excluded
 *   s_ij += bias_j
 *   out_i = softmax_j(s_ij) v_j ,  lse_i = logsumexp_j s_ij
 *
 * A row whose every entry is excluded gets the reference's value for it: the
 * uniform average of v over its keys (all keys except those both masked and
 * "dead", i.e. with bias <= -FLT_MAX/2, where the reference overflows to
 * -inf), lse = -FLT_MAX.
 *
 * Optional value multiplier (forward only): if v_mul != NULL the pass uses
 * v_j * v_mul_j as its values, so a decode step reads the order-n chain's
 * V' = v_k * msg (n_poly_attention.py:287) from the two cached tensors.
 *
 * Optional fused epilogue for the order-n chain (V' = v_k * msg,
 * n_poly_attention.py:287): if epi_out != NULL, epi_out_i = epi_mul_i * out_i is
 * written as well (same shape as out; epi_mul rows indexed like out rows).
 */
typedef struct PolyPassArgs {
  int32_t batch;
  int32_t heads;      /* query heads (q, out, lse, query-side) */
  int32_t kv_heads;   /* key/value heads (k, v, bias); divides heads */
  int32_t seq_q;
  int32_t seq_k;
  int32_t head_dim;   /* q/k/v/out feature size */
  int32_t dtype;      /* POLY_F32 / POLY_F16 / POLY_BF16 for q, k, v, out, epi_mul, epi_out */
  int32_t causal;     /* 1: key j visible to query i iff j <= i (top-left aligned) */
  float scale;        /* usually head_dim ** -0.5 */
  float softclamp;    /* > 0 enables c * tanh(s / c) */

  const void* q;        int64_t q_stride[3];     /* [batch, heads, seq_q, d]      */
  const void* k;        int64_t k_stride[3];     /* [batch, kv_heads, seq_k, d]   */
  const void* v;        int64_t v_stride[3];     /* [batch, kv_heads, seq_k, d]   */
  const void* v_mul;    int64_t v_mul_stride[3]; /* [batch, kv_heads, seq_k, d] | NULL: v_j *= v_mul_j */
  const float* bias;    int64_t bias_stride[2];  /* [batch, kv_heads, seq_k] | NULL */
  const uint8_t* key_mask;   int64_t key_mask_stride;    /* [batch, seq_k] | NULL, 0 = masked */
  const uint8_t* query_mask; int64_t query_mask_stride;  /* [batch, seq_q] | NULL, 0 = masked */
  void* out;            int64_t out_stride[3];   /* [batch, heads, seq_q, d]      */
  float* lse;           int64_t lse_stride[2];   /* [batch, heads, seq_q] | NULL  */
  const void* epi_mul;     int64_t epi_mul_stride[3];  /* [batch, heads, seq_q, d] | NULL */
  void* epi_out;           int64_t epi_out_stride[3];  /* [batch, heads, seq_q, d] | NULL */

  void* workspace;          /* device scratch, >= poly_pass_fwd_workspace_size() bytes */
  size_t workspace_bytes;

  /* With causal: key j visible to query i iff j <= i + causal_offset, i.e. the
   * queries are rows [causal_offset, causal_offset + seq_q) of a longer
   * sequence whose first seq_k keys are given (no counterpart in the
   * reference: it lets one launch cover a sequence shard's queries against
   * all earlier keys). 0 is the reference's top-left causal mask. Non-zero
   * values must be multiples of 128 and are taken by the tcgen05 forward only
   * (bf16 / fp16, head_dim 64 or 128, no masks, no softclamp); elsewhere
   * POLY_EUNSUPPORTED. Negative: POLY_EINVAL. */
  int32_t causal_offset;
  int32_t reserved_;
} PolyPassArgs;

/*
 * Backward of one pass (recomputes the scores from q, k and lse):
 *   dv_j   = sum_i p_ij dout_i
 *   ds_ij  = p_ij (dout_i . v_j - dout_i . out_i + dlse_i)
 *   dbias_j = sum_i ds_ij               (includes masked entries, as autograd does)
 *   dz_ij  = ds_ij (1 - tanh^2) on kept entries, 0 on masked ones
 *   dq_i   = scale sum_j dz_ij k_j ,   dk_j = scale sum_i dz_ij q_i
 * With GQA, dk / dv / dbias sum over the query heads of each group.
 * If dq_accumulate != 0, dq += result (used for dq2 = part1 + part2,
 * poly_attention/flash_poly_attention.py:444); otherwise dq = result.
 */
typedef struct PolyPassBwdArgs {
  PolyPassArgs fwd;         /* the forward's inputs; fwd.out and fwd.lse are required */
  const void* dout;     int64_t dout_stride[3];  /* [batch, heads, seq_q, d]    */
  const float* dlse;    int64_t dlse_stride[2];  /* [batch, heads, seq_q] | NULL */
  void* dq;             int64_t dq_stride[3];    /* [batch, heads, seq_q, d]    */
  void* dk;             int64_t dk_stride[3];    /* [batch, kv_heads, seq_k, d] */
  void* dv;             int64_t dv_stride[3];    /* [batch, kv_heads, seq_k, d] */
  float* dbias;         int64_t dbias_stride[2]; /* [batch, kv_heads, seq_k] | NULL */
  int32_t dq_accumulate;
  int32_t reserved;
  void* workspace;          /* >= poly_pass_bwd_workspace_size() bytes */
  size_t workspace_bytes;
} PolyPassBwdArgs;

/*
 * Merge P partial passes over disjoint key shards of the same queries:
 *   lse_i = logsumexp_p lse_p,i ;  out_i = sum_p exp(lse_p,i - lse_i) out_p,i
 * part_out: [P][rows][d] (dtype), part_lse: [P][rows] fp32, rows = batch*heads*seq_q
 * flattened contiguously; out: [rows][d] (dtype); lse: [rows] fp32 (may be NULL).
 */
typedef struct PolyMergeArgs {
  int32_t parts;
  int32_t head_dim;
  int32_t dtype;
  int32_t reserved;
  int64_t rows;
  const void* part_out;
  const float* part_lse;
  void* out;
  float* lse;
} PolyMergeArgs;

POLY_API int poly_pass_fwd(const PolyPassArgs* args, void* stream);
POLY_API size_t poly_pass_fwd_workspace_size(const PolyPassArgs* args);

POLY_API int poly_pass_bwd(const PolyPassBwdArgs* args, void* stream);
POLY_API size_t poly_pass_bwd_workspace_size(const PolyPassBwdArgs* args);

POLY_API int poly_lse_merge(const PolyMergeArgs* args, void* stream);

/*
 * The n passes of one KV-cache decoding step of the order-n chain, in order,
 * in one call. Contract: passes[i + 1] reads what passes[i] wrote only in the
 * LAST key row (row seq_k - 1, the row the step appended) of its v, v_mul and
 * bias; every other input is complete when the call is made (stream order);
 * no pass writes what an earlier pass of the list reads. Under it, each pass
 * after the first is launched as a programmatic dependent of the previous one:
 * its CTAs start while the previous pass drains, stream every key tile but the
 * last, and wait for the previous pass before loading the last. Every pass
 * must take the decode kernel (poly_pass_fwd_kernel_name() == "decode"), else
 * POLY_EUNSUPPORTED and nothing is launched. A pass with few (batch, kv head)
 * groups needs a workspace of poly_pass_fwd_workspace_size() bytes (0 otherwise);
 * a pass given too little gets POLY_EINVAL and nothing is launched.
 */
POLY_API int poly_decode_chain(const PolyPassArgs* passes, int n, void* stream);

/*
 * Row copies for KV-cache appends (replaces the reference's per-step
 * torch.cat cache growth, poly_attention/poly_attention.py:283-287 and
 * n_poly_attention.py:206-207, 281-302, by in-place writes of the new rows).
 * Copy i moves outer x inner rows of row_bytes bytes; row (o, i) starts at
 * src + o * src_stride[0] + i * src_stride[1] (same for dst). All n <= 16
 * copies run in ONE kernel launch. Pointers, strides and row_bytes must be
 * multiples of 16 bytes, else POLY_EINVAL.
 */
#define POLY_MAX_ROW_COPIES 16
typedef struct {
  const void* src;
  void* dst;
  int32_t outer;
  int32_t inner;
  int32_t row_bytes;
  int32_t reserved;
  int64_t src_stride[2]; /* bytes */
  int64_t dst_stride[2]; /* bytes */
} PolyRowCopy;

POLY_API int poly_copy_rows(const PolyRowCopy* copies, int n, void* stream);

/*
 * Per-head RMSNorm of query/key tensors straight from the head-split view of a
 * projection output (replaces q_norms, poly_attention/poly_attention.py:272,
 * n_poly_attention.py:186-187, and the contiguous copy torch makes of the
 * strided view first): dst = src * rsqrt(mean(src^2) + eps) * weight over the
 * last dim, fp32 arithmetic. src [batch, heads, rows, dim] with element
 * strides (batch, head, row), last dim contiguous; dst contiguous, in
 * dst_dtype (src's dtype, or F32 inside autocast). weight [dim] in
 * weight_dtype. dim <= 256, dim % 8 == 0, 16-byte aligned rows. All n <= 4
 * tensors are normalised in ONE kernel launch.
 */
#define POLY_MAX_NORMS 4
typedef struct {
  const void* src;
  void* dst;
  const void* weight;
  int32_t batch;
  int32_t heads;
  int32_t rows;
  int32_t dim;
  int64_t src_stride[3]; /* elements: batch, head, row */
  int32_t src_dtype;     /* POLY_F32 / POLY_F16 / POLY_BF16 */
  int32_t dst_dtype;
  int32_t weight_dtype;
  float eps;
} PolyHeadNorm;

POLY_API int poly_head_rmsnorm(const PolyHeadNorm* norms, int n, void* stream);

/*
 * The pass over sequences packed end to end: pass.seq_q = pass.seq_k = the
 * rows of all of them (pass.batch 1, batch strides ignored), sequence s is
 * rows [cu_seqlens[s], cu_seqlens[s + 1]) and its queries see its own keys only
 * (with causal, those at or before them). cu_seqlens is device memory: int32
 * [seqs + 1], not decreasing, within [0, seq_q]; lengths may be 0, and rows
 * outside every sequence are neither read into a result nor (without zero_rest)
 * written. Offsets
 * that break this give wrong rows, never an access outside the tensors.
 * max_len: an upper bound of the lengths if the caller has one, else 0. Up to
 * 128 it selects kernels that hold a whole sequence per CTA; all results of a
 * longer sequence are then NaN (it is not looked at otherwise). zero_rest: rows
 * outside the sequences are set to 0 in every output, but for a dq that is
 * accumulated into (seqs = 0 writes nothing). Bias, softclamp, grouped heads and
 * the epilogue product as in poly_pass_fwd; masks, v_mul and causal_offset are
 * POLY_EUNSUPPORTED. A row whose every key is dead (bias <= -FLT_MAX / 2) gets
 * out = 0 and lse = -FLT_MAX, and no gradient. epi_out is epi_mul times the
 * unrounded out.
 *
 * out_lo (optional, out's layout; 16-bit dtypes): what rounding took off out,
 * rounded itself. The backward subtracts dout . out from every entry of a row of
 * dP, so an error of out there is common to the row and does not average out
 * over the keys: given out_lo it uses out + out_lo.
 *
 * v_left, v_right (backward, optional, dv's layout): the values were the product
 * v_left * v_right (the chain's V' = v * msg). dv then receives the gradient of
 * v_left and dv_right that of v_right, each rounded once.
 */
typedef struct PolyPackedArgs {
  PolyPassArgs pass;
  const int32_t* cu_seqlens;
  int32_t seqs;
  int32_t max_len;
  int32_t zero_rest;
  int32_t reserved;
  void* out_lo;
} PolyPackedArgs;

typedef struct PolyPackedBwdArgs {
  PolyPassBwdArgs bwd;
  const int32_t* cu_seqlens;
  int32_t seqs;
  int32_t max_len;
  int32_t zero_rest;
  int32_t reserved;
  const void* out_lo;                                /* as bwd.fwd.out | NULL */
  const void* v_left;   int64_t v_left_stride[2];    /* (head, row) elements | NULL */
  const void* v_right;  int64_t v_right_stride[2];
  void* dv_right;       int64_t dv_right_stride[2];
} PolyPackedBwdArgs;

/* The workspace of the backward is 16-byte aligned. */
POLY_API int poly_packed_pass_fwd(const PolyPackedArgs* args, void* stream);
POLY_API int poly_packed_pass_bwd(const PolyPackedBwdArgs* args, void* stream);
POLY_API size_t poly_packed_pass_bwd_workspace_size(const PolyPackedBwdArgs* args);
/* "small", "tc100", "tf32x3" or "simt" ("invalid" if validation fails) */
POLY_API const char* poly_packed_pass_fwd_kernel_name(const PolyPackedArgs* args);
POLY_API const char* poly_packed_pass_bwd_kernel_name(const PolyPackedBwdArgs* args);

/*
 * Rotary positions of up to 8 query / key tensors in ONE launch. Over the
 * first rot features of a row, in pairs (a, b) = (2i, 2i + 1) (interleaved) or
 * (i, i + rot / 2):
 *   y_a = factor (x_a cos t - x_b sin t),  y_b = factor (x_b cos t + x_a sin t)
 * and y = x past rot. t = position * inv_freq[i], the product exact and reduced
 * in 64 bits, or angles[b][row][i]. inverse != 0 negates sin: the transpose,
 * which is the gradient. The tensors of a call share batch, rows, positions
 * and dtype; strides are in elements, the feature axis contiguous; dst may be
 * src with src's strides. The position of row i is pos_start plus positions
 * (int32, or int64 if pos_wide) if given, or the row's place in its sequence if
 * cu_seqlens is given (batch 1), else i.
 */
#define POLY_MAX_ROTARY 8
typedef struct {
  const void* src;
  void* dst;
  int32_t heads;
  int32_t reserved;
  int64_t src_stride[3]; /* elements: batch, head, row */
  int64_t dst_stride[3];
} PolyRotaryTensor;

typedef struct {
  int32_t batch;
  int32_t rows;
  int32_t dim;         /* <= 256 */
  int32_t rot;         /* even, 2 .. dim */
  int32_t dtype;
  int32_t interleaved;
  int32_t inverse;
  int32_t n;           /* tensors */
  float factor;        /* amplitude (1, or the long-context attention factor) */
  int32_t pos_wide;
  const void* positions;      int64_t pos_stride[2];   /* [batch, rows] | NULL; elements, 0 broadcasts */
  int64_t pos_start;
  const float* inv_freq;                               /* [rot / 2] | NULL */
  const float* angles;        int64_t angle_stride[2]; /* [batch, rows, rot / 2] | NULL */
  const int32_t* cu_seqlens;                           /* device [seqs + 1] | NULL */
  int32_t seqs;
  int32_t reserved;
  PolyRotaryTensor t[POLY_MAX_ROTARY];
} PolyRotaryArgs;

POLY_API int poly_rotary(const PolyRotaryArgs* args, void* stream);

/*
 * Decoding steps over trees of drafted tokens. Every sequence b has its own
 * number of cached tokens, lengths[b] (device int32), and a tree of `nodes` <= 64
 * drafted tokens given by parents[b][node] (device int32): the parent's index
 * (smaller than the node's own), -1 for a child of the cached tokens, or -2 for
 * a node that is padding (as are nodes below a padding node, nodes whose parent
 * index is not smaller than their own, and nodes past the capacity). A node sees
 * the cached tokens, its ancestors and itself:
 *
 *   s_ij = scale q_i . k_j (softclamp) + bias_j ;  out_i = softmax_j(s_ij) (v_j * v_mul_j)
 *
 * over the cache's rows j < lengths[b] and the rows lengths[b] + node that the
 * tree's own keys and values occupy (poly_tree_append writes them, a padding
 * node's as zeros). Padding nodes, and nodes that see dead keys only (bias
 * <= -FLT_MAX / 2), get out = 0 and lse = -FLT_MAX. Lengths are clamped to [0, capacity];
 * nothing outside the caches is ever accessed.
 *
 * out / lse take the nodes' rows; cache_out / cache_lse take them at the cache
 * rows lengths[b] + node (the next level's values and bias). Each may be NULL.
 * Everything is stream-ordered and reads lengths and parents on the device, so a
 * step can be captured in a graph and replayed.
 */
#define POLY_MAX_TREE_NODES 64
typedef struct PolyTreePass {
  int32_t batch, heads, kv_heads, nodes;
  int32_t head_dim, dtype, capacity, reserved;
  float scale, softclamp;
  const void* q;      int64_t q_stride[3];       /* [batch, heads, nodes, d]       */
  const void* k;      int64_t k_stride[3];       /* [batch, kv_heads, capacity, d] */
  const void* v;      int64_t v_stride[3];       /* [batch, kv_heads, capacity, d] */
  const void* v_mul;  int64_t v_mul_stride[3];   /* [batch, kv_heads, capacity, d] | NULL */
  const float* bias;  int64_t bias_stride[2];    /* [batch, kv_heads, capacity] | NULL */
  const int32_t* lengths;                        /* [batch] */
  const int32_t* parents; int64_t parents_stride; /* [batch, nodes], row stride */
  void* out;          int64_t out_stride[3];     /* [batch, heads, nodes, d] | NULL */
  float* lse;         int64_t lse_stride[2];     /* [batch, heads, nodes] | NULL */
  void* cache_out;    int64_t cache_out_stride[3]; /* [batch, heads, capacity, d] | NULL */
  float* cache_lse;   int64_t cache_lse_stride[2]; /* [batch, heads, capacity] | NULL */
  void* workspace;    /* >= poly_tree_workspace_size() bytes, 16-byte aligned; passes of a chain may share it */
  size_t workspace_bytes;
} PolyTreePass;

/* New rows of up to 16 caches of one shape: src [batch, kv_heads, nodes, d] to
 * cache rows lengths[b] + node. d * element size must be a multiple of 2 bytes. */
#define POLY_MAX_TREE_CACHES 16
typedef struct PolyTreeAppend {
  int32_t batch, kv_heads, nodes, row_bytes;
  int32_t capacity, n;
  const int32_t* lengths;
  const int32_t* parents; int64_t parents_stride;
  struct {
    const void* src; int64_t src_stride[3];   /* bytes: batch, head, node */
    void* cache;     int64_t cache_stride[3]; /* bytes: batch, head, row */
  } t[POLY_MAX_TREE_CACHES];
} PolyTreeAppend;

/* Keeps the accepted nodes: cache rows lengths[b] + path[b][i] move to
 * lengths[b] + i for i < count[b], then lengths[b] += count[b]. path[b] holds
 * path_len entries and ascends (a root-to-leaf path does); an entry smaller than
 * its place is taken as its place, one past the nodes as the last node; count is
 * clamped to [0, min(path_len, nodes)] and to the capacity. */
typedef struct PolyTreeCommit {
  int32_t batch, kv_heads, nodes, capacity;
  int32_t n, path_len;
  int32_t* lengths;
  const int32_t* path;  int64_t path_stride;   /* [batch, path_len], row stride */
  const int32_t* count;                        /* [batch] */
  struct {
    void* cache; int64_t cache_stride[3];      /* bytes: batch, head, row */
    int64_t row_bytes;
  } t[POLY_MAX_TREE_CACHES];
} PolyTreeCommit;

/* The append (or NULL), then n passes in order, each launched so that its CTAs
 * start while the previous kernel drains: a pass may read what an earlier one
 * wrote only in rows lengths[b] and after of its v, v_mul and bias. */
POLY_API int poly_tree_chain(const PolyTreeAppend* append, const PolyTreePass* passes, int n, void* stream);
POLY_API size_t poly_tree_workspace_size(const PolyTreePass* pass);
POLY_API int poly_tree_commit(const PolyTreeCommit* args, void* stream);
/* The same with the nodes of the last step kept on the device, where a replayed
 * step counts too: the append writes its nodes to *step_nodes (device int32), and
 * the commit takes min(*step_nodes, nodes) for nodes, then sets *step_nodes to 0,
 * so that a second commit keeps nothing. NULL: as above. */
POLY_API int poly_tree_chain_counted(const PolyTreeAppend* append, const PolyTreePass* passes, int n, int32_t* step_nodes,
                                     void* stream);
POLY_API int poly_tree_commit_counted(const PolyTreeCommit* args, int32_t* step_nodes, void* stream);
/* positions[b][node] = lengths[b] + the node's ancestors in the tree (rotary
 * positions of the drafted tokens); lengths[b] for padding. */
POLY_API int poly_tree_positions(const int32_t* lengths, const int32_t* parents, int64_t parents_stride, int batch,
                                 int nodes, int32_t* positions, int64_t positions_stride, void* stream);
/* "tree" (mma.sync), "tc100" (tcgen05: more than 32 rows per key) or "simt"; "invalid" if validation fails */
POLY_API const char* poly_tree_kernel_name(const PolyTreePass* pass);

/*
 * poly_pass_bwd without a caller workspace. No counterpart in the reference:
 * it exists for callers that cannot allocate device memory (FFI hosts that
 * only pass existing buffers, processes whose device memory another
 * allocator has fully planned). Scratch comes from an 8 MiB array built into
 * the library (held per GPU until exit); larger problems get POLY_EINVAL.
 * All calls on a device share that array: calls overlapping on the GPU race.
 * Every call outside stream capture resolves the array's address afresh
 * (a device reset leaves no stale address); a call during capture reuses the
 * last one, so make the first call on a device before any stream capture.
 * args->workspace is ignored.
 */
POLY_API int poly_pass_bwd_noalloc(const PolyPassBwdArgs* args, void* stream);
POLY_API size_t poly_noalloc_scratch_bytes(void);

/* Name of the kernel family poly_pass_fwd / poly_pass_bwd would launch for
 * these arguments: forward "decode" (one query row against a cache), "small"
 * (short sequences, mma.sync), "tf32x3" (fp32 on tensor cores), "tc100"
 * (tcgen05) or "simt" (CUDA cores); backward "tc100" or "simt"; "invalid"
 * when the arguments fail validation. */
POLY_API const char* poly_pass_fwd_kernel_name(const PolyPassArgs* args);
POLY_API const char* poly_pass_bwd_kernel_name(const PolyPassBwdArgs* args);

/* Last error message of the calling thread ("" if none). */
POLY_API const char* poly_last_error(void);

/* Number of kernels this library has launched in this process. */
POLY_API unsigned long long poly_launch_count(void);

/* Device error word of the current device (synchronous read): non-zero if a
 * kernel's bounded wait gave up since the last reset: 1 | site << 8, the
 * first give-up wins. The launch that gave up freed its resources and
 * returned; the outputs of that call are undefined. Other CTAs of the same
 * launch give up at once; later launches run normally whether or not the
 * word has been reset. reset != 0 clears the word. */
POLY_API int poly_device_error(int* out, int reset);

/* Diagnostics, no counterpart in the reference: launches one CTA that holds
 * TMEM and waits on a barrier nothing arrives on, with a wait limit of
 * limit_ns (0 < limit_ns <= 1e9), so the bounded-wait give-up path runs:
 * *result (device int) becomes 2 once the wait gave up and the CTA freed its
 * TMEM and returned (1 if the wait wrongly succeeded); the device error word
 * then reads 1 | 99 << 8. */
POLY_API int poly_selftest_wait_timeout(unsigned long long limit_ns, int* result, void* stream);

/* ABI checks for bindings: POLY_ABI_VERSION and the struct sizes. */
POLY_API int poly_abi_version(void);
POLY_API size_t poly_sizeof_pass_args(void);
POLY_API size_t poly_sizeof_pass_bwd_args(void);
POLY_API size_t poly_sizeof_merge_args(void);
POLY_API size_t poly_sizeof_rotary_args(void);
POLY_API size_t poly_sizeof_packed_args(void);
POLY_API size_t poly_sizeof_tree_pass(void);
POLY_API size_t poly_sizeof_tree_append(void);
POLY_API size_t poly_sizeof_tree_commit(void);
POLY_API size_t poly_sizeof_packed_bwd_args(void);

#ifdef __cplusplus
}
#endif

#endif /* POLY_ATTENTION_H_ */
