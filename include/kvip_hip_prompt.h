/*
 * kvip_hip_prompt.h - C ABI of the operators on either side of a prompt chunk's layers
 * (libkvip_hip.so): attention of a chunk over the paged cache, queries and keys normed and turned
 * (and quantised for the indexer), logits turned into the probabilities that tokens are drawn from.
 *
 * The conventions are those of kvip_hip.h and kvip_hip_draft.h: plain pointers and sizes, a
 * hipStream_t passed as void*, calls that only enqueue (no allocation, synchronisation, memset or
 * read-back, so each can be captured into a hipGraph), KVIP_ERR_INVALID for arguments rejected
 * before anything is launched, device-side problems OR-ed into an optional status word; packed
 * steps: request b's rows are cu_seqlens[b] .. cu_seqlens[b + 1]. There is no counterpart in the
 * reference, whose service leaves these steps to its engine.
 */
#ifndef KVIP_HIP_PROMPT_H
#define KVIP_HIP_PROMPT_H

#include "kvip_hip_draft.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KVIP_PROMPT_ABI_VERSION 1u

#define KVIP_NORM_NONE 0
#define KVIP_NORM_RMS 1             /* x / sqrt(mean x^2 + epsilon) */
#define KVIP_NORM_LAYER 2           /* (x - mean x) / sqrt(mean (x - mean x)^2 + epsilon) */

#define KVIP_NORM_MAX_DIM 512
#define KVIP_LOGIT_MAX_BIASES 4096

/* Attention of a chunk of new tokens over the paged rows of its request, of which seq_lens[b] are there,
 * the last n = cu_seqlens[b + 1] - cu_seqlens[b] those of the chunk. Token i sees the rows of positions
 * 0 .. seq_lens[b] - n + i. Keys and values as for kvip_hip_sparse_attention; per token and head
 *   output = sum_j p_j value_j / sum_j p_j, p_j = exp(s_j - max s), s_j = scale <query, key_j>
 * over the rows it sees (0 where it sees none), lse = log sum_j exp(s_j) (-infinity).
 * Features times their scales (products in 32 bits) are rounded once to fp16 under an exponent that the rows of 32
 * positions share, their largest feature being 2^11 .. 2^15 there: by 2^-11 of themselves, or 2^-36 of that largest;
 * rows whose largest features are more than 2^12 apart stand under exponents of their own; query features likewise, which
 * only those below 2^-28 of the largest of their (token, head) feel; probabilities by 2^-11 of themselves, or, for an
 * output, by 2^-36 of the largest feature that the token sees. The rest is in 32 bits.
 * Rows that a token does not see do not reach its output, whatever they hold; a token that sees a row with
 * a value that is no finite 32-bit number becomes NaN as a whole (a rotary feature that is not finite reaches the
 * logits as it is). Blocks outside the cache set KVIP_STATUS_BAD_BLOCK and
 * count as not there; lengths outside 0 .. max_blocks * 128, fewer rows than chunk tokens, or cu_seqlens that
 * fall or leave 0 .. max_tokens set KVIP_STATUS_BAD_LENGTH (they are cut to the range; a row of several requests goes with
 * the first of them, but where kvip_hip_tree_attention does the work, see below). So does a request
 * whose rows and those of the requests before it, each request's rounded up to 32, are more than max_rows rounded up
 * to 32 plus 32 * batch: it sees nothing. With steps, a request with steps[b] <= 0 (one that
 * kvip_hip_page_tables_extend refused) sees nothing: output 0, lse -infinity. Rows of output and lse behind
 * cu_seqlens[batch] are left as they were. A workspace serves one call at a time, and the lengths stay as
 * they are while it runs.
 * Where max_tokens is at most 64 and max_tokens * heads at most 512 * batch, kvip_hip_tree_attention does the work
 * (without visible): it rounds probabilities times scales to bf16 (2^-8), not features, holds weighted sums of values as they are
 * (which values of 10^35 and more on some rows take past 32 bits), and max_rows does not count. Elsewhere the workspace has 1152
 * bytes for each of max_rows and of 32 rows per request, and 269 MB for the parts of contexts that are cut. */
typedef struct KvipChunkAttnArgs {
    const uint16_t* query;        /* [max_tokens, heads, 576] bf16, 16-byte aligned */
    const uint8_t* kv_cache;      /* 16-byte aligned */
    const int32_t* block_table;   /* [batch, max_blocks] */
    const int32_t* seq_lens;      /* [batch] */
    const int32_t* cu_seqlens;    /* [batch + 1], at most max_tokens */
    const int32_t* steps;         /* [batch], or NULL */
    void* output;                 /* [max_tokens, heads, 512], 16-byte aligned */
    float* lse;                   /* [max_tokens, heads], or NULL */
    void* workspace;              /* kvip_hip_chunk_attention_workspace_bytes bytes, 16-byte aligned */
    uint32_t* status;             /* optional */
    int64_t kv_block_stride;      /* bytes, >= 128 * row_stride, multiple of 16 */
    int64_t max_rows;             /* cached rows of all requests together that the workspace is for, 1..2^31 */
    int32_t row_stride;           /* bytes, 656..2^24, multiple of 16 */
    int32_t batch;                /* 1..KVIP_DRAFT_MAX_BATCH */
    int32_t heads;                /* 1..128 */
    int32_t max_tokens;           /* 1..KVIP_DRAFT_MAX_TOKENS */
    int32_t max_blocks;           /* 1..2^17, as the workspace's */
    int32_t num_blocks;           /* 1..2^24 - 1 */
    int32_t output_dtype;         /* KVIP_DTYPE_BF16 or _FP32 */
    float scale;                  /* finite */
} KvipChunkAttnArgs;

/* Norm of every head over its dim features, times weight, plus bias (each optional), then the first
 * rotary_dim features turned as by kvip_hip_rotary. In 32 bits (the angle's turns in 64), rounded once.
 * Up to two arrays a call: tensors[0] the queries, tensors[1] the keys. strides in elements, the last dimension
 * contiguous; an output is its input's array with the same strides, or does not overlap it.
 *
 * Quantised (`quantised`: queries and keys both, dim 128): each head of a query gets a scale, its largest magnitude /
 * 448 (1 where that quotient is 0), and e4m3 features rounded from feature / scale; a NaN stays one and does not
 * count for the scale, an infinity makes the scale infinite and itself a NaN. Keys have one head;
 * token t's goes to slot slots[t] of the paged index cache (negative: none; past the cache:
 * KVIP_STATUS_BAD_TOKEN and none). Slots of one call differ. */
typedef struct KvipNormTensor {
    const void* x;                /* [tokens, heads, dim], NULL: none */
    void* out;                    /* as x; quantised: bytes, of keys [num_blocks, 128, 128] */
    const float* weight;          /* [dim], or NULL */
    const float* bias;            /* [dim], or NULL */
    float* scales;                /* quantised: [tokens, heads], of keys [num_blocks, 128] */
    int64_t x_token, x_head;
    int64_t out_token, out_head;  /* of quantised keys: bytes from block to block, floats from block to block of scales */
    int32_t heads;
    int32_t norm;                 /* KVIP_NORM_* */
} KvipNormTensor;

typedef struct KvipNormRotaryArgs {
    KvipNormTensor tensors[2];
    const int64_t* positions;     /* [tokens] */
    const double* frequencies;    /* [rotary_dim / 2], radians per position */
    const int64_t* slots;         /* quantised, with keys: [tokens] */
    uint32_t* status;             /* optional */
    int64_t tokens;
    int32_t dim;                  /* rotary_dim..KVIP_NORM_MAX_DIM; quantised: 128 */
    int32_t rotary_dim;           /* even, 2.. */
    int32_t half;                 /* 1: halves, 0: interleaved pairs */
    int32_t dtype;                /* of x (and of out): KVIP_DTYPE_BF16, _FP16 or _FP32 */
    int32_t quantised;
    int32_t num_blocks;           /* of the index cache */
    float epsilon;                /* >= 0, finite */
    float magnitude;
} KvipNormRotaryArgs;

/* What requests hold already: counts[b][v] = how often request b wrote token v, bit v % 32 of
 * seen[b][v / 32] = it wrote v or its prompt has it.
 *
 * kvip_hip_history_load replaces request requests[i]'s (negative: none) by tokens cu_seqlens[i] ..
 * cu_seqlens[i + 1], of which the first prompt_lens[i] are its prompt. Requests of one call differ.
 * kvip_hip_history_append adds the first kept[b] of tokens[b] (as kvip_hip_verify_drafts writes them).
 * Tokens outside 0 .. vocab - 1 set KVIP_STATUS_BAD_TOKEN and are left out; requests outside 0 .. batch - 1,
 * cu_seqlens that fall or leave 0 .. max_tokens and kept outside 0 .. token_stride set KVIP_STATUS_BAD_LENGTH
 * (such a request is left out, the others are cut to the range). */
typedef struct KvipHistoryArgs {
    int32_t* counts;              /* [batch, vocab] */
    uint32_t* seen;               /* [batch, (vocab + 31) / 32] */
    const int64_t* tokens;        /* load: [max_tokens]; append: [batch, token_stride] */
    const int32_t* requests;      /* load: [count] */
    const int32_t* cu_seqlens;    /* load: [count + 1] */
    const int32_t* prompt_lens;   /* load: [count] */
    const int32_t* kept;          /* append: [batch] */
    uint32_t* status;             /* optional */
    int64_t max_tokens;           /* load: 0..2^31 - 1 */
    int32_t count;                /* load: requests, 1..KVIP_DRAFT_MAX_BATCH */
    int32_t batch;                /* 1..KVIP_DRAFT_MAX_BATCH */
    int32_t vocab;                /* 1..2^20 */
    int32_t token_stride;         /* append: 1..KVIP_DRAFT_MAX_NODES */
} KvipHistoryArgs;

/* Probabilities of the next token from logits, row by row of a packed step. With n how often the request
 * wrote token v (counts, read for the tokens of seen alone, and the row's ancestors among the step's tokens 1 .. 63:
 * bit i of visible[row] names token i, token 0 being in the history already; without visible, as for the last rows of
 * prompt chunks, there are none) and x the logit in 32 bits:
 *   x = x > 0 ? x / repetition : x * repetition   where the request holds v (seen, or an ancestor);
 *   x = x - presence - frequency * n              where n > 0;
 *   x = x + the biases of v in the request's list (in the list's order; token negative: none);
 *   x = -infinity                                 where bit v % 32 of allowed[row][v / 32] is 0;
 *   probs = exp((x - max x) / temperature) / their sum, or, where temperature is not above 0, 1 at the first of the
 *   largest x and 0 elsewhere.
 * Each array is optional (repetition 1, the others 0, temperature 1). In 32 bits; where temperature is above 0, x / repetition may
 * be x times the rounded reciprocal, where it is not, numbers that are 32-bit ones stay exact, so that tokens tie. Sums are 32-bit, over at most 2^17 terms per
 * run and then over the runs; probabilities are rounded once. An x that is NaN counts as -infinity and sets
 * KVIP_STATUS_BAD_PROBS, as does a row that is -infinity everywhere, which gets 0 everywhere; tokens at +infinity
 * share the row. Drafted or bias tokens past vocab - 1 (drafted: or negative) set KVIP_STATUS_BAD_TOKEN and are left out;
 * cu_seqlens that fall or leave 0 .. max_tokens set KVIP_STATUS_BAD_LENGTH (a row goes with the first request that
 * holds it). Rows of no request are left as they were. Where max_tokens rows would take more workgroups than a
 * launch has, workspace_bytes is 0 and the call is refused. */
typedef struct KvipLogitArgs {
    const void* logits;           /* [max_tokens, vocab], rows logits_stride elements apart */
    void* probs;                  /* [max_tokens, vocab], rows probs_stride apart, not the logits' memory */
    const int32_t* cu_seqlens;    /* [batch + 1] */
    const float* temperature;     /* [batch], or NULL; so the next three */
    const float* repetition;
    const float* presence;
    const float* frequency;
    const int32_t* counts;        /* [batch, vocab], with seen; or NULL */
    const uint32_t* seen;         /* [batch, (vocab + 31) / 32] */
    const int64_t* tokens;        /* [max_tokens], with visible; or NULL */
    const int64_t* visible;       /* [max_tokens] */
    const int32_t* bias_tokens;   /* [batch, biases], with bias_values; or NULL */
    const float* bias_values;
    const uint32_t* allowed;      /* [max_tokens, (vocab + 31) / 32], or NULL */
    void* workspace;              /* kvip_hip_process_logits_workspace_bytes bytes, 16-byte aligned; one call at a time */
    uint32_t* status;             /* optional */
    int64_t logits_stride, probs_stride;
    int32_t batch;                /* 1..KVIP_DRAFT_MAX_BATCH */
    int32_t max_tokens;           /* 1..KVIP_DRAFT_MAX_TOKENS */
    int32_t vocab;                /* 1..2^20 */
    int32_t biases;               /* 0..KVIP_LOGIT_MAX_BIASES */
    int32_t dtype;                /* of logits: KVIP_DTYPE_FP32, _BF16 or _FP16 */
    int32_t probs_dtype;          /* the same */
} KvipLogitArgs;

uint32_t kvip_hip_prompt_abi_version(void);
uint32_t kvip_hip_chunk_attention(const KvipChunkAttnArgs* args, void* stream);
uint64_t kvip_hip_chunk_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t max_tokens, int32_t max_blocks, int64_t max_rows);
uint32_t kvip_hip_norm_rotary(const KvipNormRotaryArgs* args, void* stream);
uint32_t kvip_hip_history_load(const KvipHistoryArgs* args, void* stream);
uint32_t kvip_hip_history_append(const KvipHistoryArgs* args, void* stream);
uint32_t kvip_hip_process_logits(const KvipLogitArgs* args, void* stream);
uint64_t kvip_hip_process_logits_workspace_bytes(int32_t max_tokens, int32_t vocab);

#ifdef __cplusplus
}
#endif

#endif /* KVIP_HIP_PROMPT_H */
