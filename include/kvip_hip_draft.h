/*
 * kvip_hip_draft.h - C ABI of the operators of a round of drafted tokens (libkvip_hip.so):
 * page tables and slot maps, rotary positions, the rows of the paged KV cache, attention of a
 * tree of drafted tokens over that cache, verification of the drafted tokens.
 *
 * The conventions are those of kvip_hip.h: plain pointers and sizes, a hipStream_t passed as
 * void*, calls that only enqueue (no allocation, synchronisation, memset or read-back, so each
 * can be captured into a hipGraph), KVIP_ERR_INVALID for arguments rejected before anything is
 * launched, device-side problems OR-ed into an optional status word. There is no counterpart
 * in the reference, whose service leaves these steps to its engine.
 *
 * A step is packed: request b's tokens are rows cu_seqlens[b] .. cu_seqlens[b + 1] of every
 * per-token array. Token 0 of a request is its last committed token (or any other token that is
 * not drafted); the others are drafted. parents[row] names a token's parent within its request
 * (-1: none; a parent comes before its children). Without parents each token's parent is the
 * one before it (a chain).
 */
#ifndef KVIP_HIP_DRAFT_H
#define KVIP_HIP_DRAFT_H

#include "kvip_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KVIP_DRAFT_ABI_VERSION 2u

/* Device status bits beside those of kvip_hip.h (BAD_BLOCK 1, HISTOGRAM 2, BAD_TOKEN 4). */
#define KVIP_STATUS_NO_PAGE 8u      /* a request got no pages: the free list is too short */
#define KVIP_STATUS_BAD_LENGTH 16u  /* a length or count outside its range */
#define KVIP_STATUS_BAD_TREE 32u    /* a parent that does not come before its child, or a path that does not rise */
#define KVIP_STATUS_BAD_PROBS 64u   /* no token can be drawn: a row without a weight, or whose weights have no finite sum */

#define KVIP_DTYPE_FP16 3           /* beside the KVIP_DTYPE_* of kvip_hip.h */

#define KVIP_DRAFT_MAX_NODES 64     /* step tokens of a request with visibility bits */
#define KVIP_DRAFT_MAX_BATCH 1024
#define KVIP_DRAFT_MAX_TOKENS (1 << 20)

/* A paged cache whose rows kvip_hip_page_tables_move copies: row of slot s (block s / 128, s % 128)
 * at base + (s / 128) * block_stride + (s % 128) * row_stride. All in bytes, multiples of 4; no row
 * lies over another. */
typedef struct KvipPagedRows {
    int64_t base;
    int64_t block_stride;
    int64_t row_stride;
    int64_t row_bytes;
} KvipPagedRows;

/* Page tables of a batch and the layout of its next step.
 *
 * State: block_table[b][j] = page of positions 128 j .. + 127 of request b (-1 past its pages),
 * lengths[b] tokens, and the free pages as a stack free_pages[0 .. free_count).
 *
 * kvip_hip_page_tables_extend appends counts[b] tokens to every request. Pages are popped in request
 * order. A request is refused, and keeps its length, where its count is negative or takes it past
 * max_blocks * 128 positions, where its rows would pass max_tokens, where it has parents and more
 * than 64 tokens (KVIP_STATUS_BAD_LENGTH), or where it and the requests before it need more pages
 * than there are (KVIP_STATUS_NO_PAGE; one that needs none is not refused for that). Writes
 *   cu_seqlens[b]   = sum of the counts before b (a negative one counts as 0), at most max_tokens;
 *   bases[b]        = the length before; steps[b] = the tokens appended (0: refused; a refused request
 *                     keeps its rows in the step, so what reads these needs steps as well);
 *   slots[row]      = page * 128 + position % 128 of the token, -1 for refused requests and for
 *                     rows behind the last token;
 *   positions[row]  = length before + depth in the tree (chain: + place); rows behind: 0;
 *   visible[row]    bit i: step token i of the request is this token or one of its ancestors
 *                     (chain: bits 0 .. place, at most all 64); rows behind: 0.
 *
 * kvip_hip_page_tables_truncate cuts every request to a shorter length, clears the table entries of the
 * pages that are no longer needed and pushes those, in the order that undoes their popping:
 * lengths[b] = clamp(targets[b], 0, lengths[b]) where `kept` is 0, else (kept: the first targets[b]
 * tokens of the step, at most steps[b]) lengths[b] = bases[b] + targets[b]. Afterwards bases[b] =
 * lengths[b], steps[b] = 0.
 *
 * kvip_hip_page_tables_move copies the rows of the kept tokens together, before a truncate with
 * `kept`: for i < targets[b], position bases[b] + i gets the rows of position bases[b] +
 * path[b][i], in `row_sets` caches. A path rises strictly and stays below steps[b], else the
 * copying of that request stops there and KVIP_STATUS_BAD_TREE is set. A target above path_stride
 * sets KVIP_STATUS_BAD_LENGTH: rows past the path's places stay where they are. */
typedef struct KvipPageTableArgs {
    int32_t* block_table;         /* [batch, max_blocks] */
    int32_t* lengths;             /* [batch] */
    int32_t* free_pages;          /* [num_blocks] */
    int32_t* free_count;          /* [1] */
    int32_t* bases;               /* [batch] */
    int32_t* steps;               /* [batch] */
    int32_t* ticket;              /* [1], 0 between calls */
    const int32_t* counts;        /* extend: [batch] */
    const int32_t* parents;       /* extend: [max_tokens], or NULL */
    const int32_t* targets;       /* truncate, move: [batch] */
    const int32_t* path;          /* move: [batch, path_stride] */
    const KvipPagedRows* rows;    /* move: device array of row_sets caches */
    int32_t* cu_seqlens;          /* extend: [batch + 1] */
    int64_t* positions;           /* extend: [max_tokens] */
    int64_t* slots;               /* extend: [max_tokens] */
    int64_t* visible;             /* extend: [max_tokens]; without parents NULL leaves it out */
    uint32_t* status;             /* optional */
    int32_t batch;                /* 1..KVIP_DRAFT_MAX_BATCH */
    int32_t max_blocks;
    int32_t num_blocks;
    int32_t max_tokens;           /* 1..KVIP_DRAFT_MAX_TOKENS */
    int32_t path_stride;
    int32_t row_sets;
    int32_t kept;
    int32_t reserved;
} KvipPageTableArgs;

/* Rotary positions: features of pair i (interleaved: 2 i and 2 i + 1; halves: i and rotary_dim / 2 + i)
 * of the first rotary_dim features of every head become
 *   (a cos - b sin, b cos + a sin) * magnitude,  angle = positions[token] * frequencies[i],
 * the angle's turns in 64 bits, the rest in 32, rounded once. `inverse` turns by the negative angle.
 * The features behind the first rotary_dim are copied where the output is another array. Up to two
 * arrays a call; strides in elements, the last dimension contiguous; an output is its input's
 * array with the same strides, or does not overlap it. */
typedef struct KvipRotaryTensor {
    const void* x;                /* [tokens, heads, dim], NULL: none (heads 0) */
    void* out;
    int64_t x_token, x_head;
    int64_t out_token, out_head;
    int32_t heads;
    int32_t dim;                  /* >= rotary_dim */
} KvipRotaryTensor;

typedef struct KvipRotaryArgs {
    KvipRotaryTensor tensors[2];
    const int64_t* positions;     /* [tokens] */
    const double* frequencies;    /* [rotary_dim / 2], radians per position */
    int64_t tokens;
    int32_t rotary_dim;           /* even, 2..512 */
    int32_t half;                 /* 1: halves, 0: interleaved pairs */
    int32_t inverse;
    int32_t dtype;                /* KVIP_DTYPE_BF16, _FP16 or _FP32 */
    float magnitude;
    int32_t reserved;
} KvipRotaryArgs;

/* Rows of the paged KV cache (656 bytes: 512 fp8 e4m3 features, 64 bf16 rotary features, four fp32
 * scales). Token t's row goes to slot slots[t] (negative: none; past the cache: KVIP_STATUS_BAD_TOKEN
 * and none): for each 128 latent features scale = largest magnitude / 448 (1 where that quotient is 0) and
 * features rounded from latent / scale. A NaN stays one and does not count for the scale; an infinity makes its
 * group's scale infinite and itself a NaN. The rotary features turned as above (positions given) or
 * as they are (NULL). Slots of one call differ. */
typedef struct KvipRowStoreArgs {
    const void* latent;           /* [tokens, 512], rows latent_stride elements apart */
    const void* rope;             /* [tokens, 64], rows rope_stride elements apart */
    const int64_t* slots;         /* [tokens] */
    const int64_t* positions;     /* [tokens], or NULL */
    const double* frequencies;    /* [32], with positions */
    uint8_t* kv_cache;            /* 16-byte aligned */
    uint32_t* status;             /* optional */
    int64_t latent_stride, rope_stride;
    int64_t kv_block_stride;      /* bytes, >= 128 * row_stride, multiple of 16 */
    int64_t tokens;
    int32_t row_stride;           /* bytes, >= 656, multiple of 16 */
    int32_t num_blocks;
    int32_t half;
    int32_t dtype;                /* of latent and rope: KVIP_DTYPE_BF16, _FP16 or _FP32 */
    float magnitude;
    int32_t reserved;
} KvipRowStoreArgs;

/* Attention of every step token over the paged rows of its request, of which seq_lens[b] are there,
 * the last ones those of its n = cu_seqlens[b + 1] - cu_seqlens[b] step tokens. Token i sees every
 * row before them and, of them, row j where bit j of visible[row] is set (visible NULL: j <= i).
 * Keys and values as for kvip_hip_sparse_attention; per token and head
 *   output = sum_j p_j value_j / sum_j p_j, p_j = exp(s_j - max s), s_j = scale <query, key_j>
 * over the rows it sees (0 where it sees none), lse = log sum_j exp(s_j) (-infinity).
 * Probabilities times a group's scale are rounded once to bf16; the rest is exact or in 32 bits.
 * Rows that a token does not see do not reach its output, whatever they hold; a token that sees a row with a
 * NaN or a scale that is not finite becomes NaN as a whole. Blocks outside the cache set
 * KVIP_STATUS_BAD_BLOCK and count as not there; lengths outside 0 .. max_blocks * 128, fewer
 * rows than step tokens, more than max_nodes of these, or cu_seqlens that fall or leave 0 .. max_tokens
 * set KVIP_STATUS_BAD_LENGTH (lengths and rows are cut to the range, tokens past max_nodes are not
 * computed). With steps, a request with steps[b] <= 0 (one that kvip_hip_page_tables_extend refused) sees
 * nothing: output 0, lse -infinity. Rows of output and lse behind cu_seqlens[batch] are left as they were.
 * The launch counts steps of 32 rows x 128 (token, head) pairs in 32 bits: where batch * heads *
 * max_nodes * max_blocks could pass that, workspace_bytes is 0 and the call is refused. A workspace serves
 * one call at a time, and the lengths stay as they are while it runs. */
typedef struct KvipTreeAttnArgs {
    const uint16_t* query;        /* [max_tokens, heads, 576] bf16, 16-byte aligned */
    const uint8_t* kv_cache;      /* 16-byte aligned */
    const int32_t* block_table;   /* [batch, max_blocks] */
    const int32_t* seq_lens;      /* [batch] */
    const int32_t* cu_seqlens;    /* [batch + 1], at most max_tokens */
    const int64_t* visible;       /* [max_tokens], or NULL */
    void* output;                 /* [max_tokens, heads, 512], 16-byte aligned */
    float* lse;                   /* [max_tokens, heads], or NULL */
    void* workspace;              /* kvip_hip_tree_attention_workspace_bytes bytes, 16-byte aligned */
    uint32_t* status;             /* optional */
    int64_t kv_block_stride;      /* bytes, >= 128 * row_stride, multiple of 16 */
    int32_t row_stride;           /* bytes, 656..2^24, multiple of 16 */
    int32_t batch;                /* 1..KVIP_DRAFT_MAX_BATCH */
    int32_t heads;                /* 1..128 */
    int32_t max_nodes;            /* 1..KVIP_DRAFT_MAX_NODES */
    int32_t max_tokens;
    int32_t max_blocks;           /* 1..2^17 */
    int32_t num_blocks;
    int32_t output_dtype;         /* KVIP_DTYPE_BF16 or _FP32 */
    float scale;                  /* finite */
    int32_t reserved;
    const int32_t* steps;         /* [batch], or NULL */
} KvipTreeAttnArgs;

/* Verification of drafted tokens. probs[row][v] is the target's probability of token v after the
 * row's token, which follow from its logits as the sampler wants them and sum to 1. A walk starts at
 * a request's token 0 and moves from a token to one of its children or ends there:
 *   chain with draft_probs (draft_probs[row] = what the next row's token was drawn from): the child x
 *     is taken where uniforms[row] * draft_probs[row][x] < probs[row][x];
 *   otherwise (tokens chosen, not drawn): the children x_1, x_2, ... in row order are taken where
 *     uniforms[row] falls into [0, p(x_1)), [p(x_1), p(x_1) + p(x_2)), ... (a token named again has 0).
 * Where the walk ends, one more token is drawn, the first v at which the running sum of the weights
 * passes final_uniforms[b] times their whole: weights max(probs - draft_probs, 0) after a
 * refused child of a chain with draft_probs, else probs without the children's tokens. Sums in 64 bits.
 * So a token is distributed as the target says, whatever was drafted. Probabilities of few bits need not sum to
 * 1: where nothing has a weight, probs are drawn from after a refused child of a chain with draft_probs, and
 * else the last child that has a probability is the token drawn.
 *   path[b]          rows (within the request) of the walk, kept[b] of them, then -1;
 *   out_tokens[b]    the walk's tokens after token 0, then the drawn one, then -1.
 * A request without rows gets kept 0, as does, with steps, one with steps[b] <= 0 (which
 * kvip_hip_page_tables_extend refused). Tokens outside 0 .. vocab - 1 set KVIP_STATUS_BAD_TOKEN and are never
 * taken; parents that do not come before their child set KVIP_STATUS_BAD_TREE and count as -1; a
 * request of more than max_nodes rows (the rest is not looked at) and cu_seqlens that fall or leave
 * 0 .. max_tokens (cut to it) set KVIP_STATUS_BAD_LENGTH; a row in which no token has a weight, or the
 * weights no finite sum, sets KVIP_STATUS_BAD_PROBS and gives token -1. Weights that are negative or NaN
 * count as 0. */
typedef struct KvipVerifyArgs {
    const void* probs;            /* [max_tokens, vocab], rows probs_stride elements apart */
    const void* draft_probs;      /* the same, draft_stride; or NULL */
    const int64_t* tokens;        /* [max_tokens] */
    const int32_t* cu_seqlens;    /* [batch + 1] */
    const int32_t* parents;       /* [max_tokens], or NULL (a chain); NULL with draft_probs */
    const float* uniforms;        /* [max_tokens], in [0, 1) */
    const float* final_uniforms;  /* [batch], in [0, 1) */
    int64_t* out_tokens;          /* [batch, max_nodes] */
    int32_t* kept;                /* [batch] */
    int32_t* path;                /* [batch, max_nodes] */
    void* workspace;              /* kvip_hip_verify_drafts_workspace_bytes bytes, 8-byte aligned, zero before its first call;
                                     calls of other shapes may follow in it, one at a time */
    uint32_t* status;             /* optional */
    int64_t probs_stride, draft_stride;
    int32_t batch;                /* 1..KVIP_DRAFT_MAX_BATCH */
    int32_t max_nodes;            /* 1..KVIP_DRAFT_MAX_NODES */
    int32_t max_tokens;
    int32_t vocab;                /* 1..2^20 */
    int32_t dtype;                /* of probs and draft_probs: KVIP_DTYPE_FP32, _BF16 or _FP16 */
    int32_t reserved;
    const int32_t* steps;         /* [batch], or NULL */
} KvipVerifyArgs;

uint32_t kvip_hip_draft_abi_version(void);
uint32_t kvip_hip_page_tables_extend(const KvipPageTableArgs* args, void* stream);
uint32_t kvip_hip_page_tables_move(const KvipPageTableArgs* args, void* stream);
uint32_t kvip_hip_page_tables_truncate(const KvipPageTableArgs* args, void* stream);
uint32_t kvip_hip_rotary(const KvipRotaryArgs* args, void* stream);
uint32_t kvip_hip_store_rows(const KvipRowStoreArgs* args, void* stream);
uint32_t kvip_hip_tree_attention(const KvipTreeAttnArgs* args, void* stream);
uint64_t kvip_hip_tree_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t max_nodes, int32_t max_blocks);
uint32_t kvip_hip_verify_drafts(const KvipVerifyArgs* args, void* stream);
uint64_t kvip_hip_verify_drafts_workspace_bytes(int32_t batch, int32_t vocab);

#ifdef __cplusplus
}
#endif

#endif /* KVIP_HIP_DRAFT_H */
