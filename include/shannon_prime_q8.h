/*
 * shannon_prime_q8.h — the 8-bit tier of the KV cache (sm_100a): rotary
 * positions with several axes, a cache held in 8 bits with one scale for
 * each block of tokens and head, its quantising write and its read back, and
 * attention over it for prompts, chunks, draft tokens and single tokens of a
 * batch of sequences.
 *
 * No counterpart in the reference, whose fp8 bands are advisory
 * (shannon_prime_llama.c:287-326) and whose attention runs in ggml.  The
 * conventions are those of shannon_prime_cuda.h: device pointers are plain
 * addresses, a stream is a cudaStream_t passed as void*, every entry point
 * returns SP_OK or an SP_ERR_* code (sp_cuda_last_error_string() has the
 * message), work is stream-ordered, nothing is allocated after
 * sp_cuda_q8_cache_init, nothing synchronises the stream unless it says so,
 * and every call but the initialisers can be captured in a CUDA graph.
 *
 * The order of one layer's step:
 *     sp_cuda_rope_axes          q and k of the new tokens, in place or not
 *     sp_cuda_q8_write_kv_tokens their k and v into the cache
 *     sp_cuda_q8_attn            their q against everything that is cached
 */
#ifndef SHANNON_PRIME_Q8_H
#define SHANNON_PRIME_Q8_H

#include <stddef.h>
#include <stdint.h>

#include "shannon_prime_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------- rotary positions -- */

#define SP_ROPE_MAX_AXES 4

/* Which elements of a head's first rot_dim make a pair. */
#define SP_ROPE_ADJACENT 0   /* (2i, 2i+1) */
#define SP_ROPE_HALVES   1   /* (i, i + rot_dim/2) */

/* Flags of sp_rope_axes_init. */
#define SP_ROPE_INTERLEAVED 1 /* pairs go to the axes in turn (an axis whose section is used up
                                 is passed over); without it each axis has a run of pairs */
#define SP_ROPE_AXIS_LADDER 2 /* the frequencies start again in each axis:
                                 theta^(-j/sections[a]) for its j-th pair; without it
                                 theta^(-2i/rot_dim) for pair i whatever its axis */

/* A rotation plan: plain host data, filled by sp_rope_axes_init and free to
 * be copied. */
typedef struct {
    int      head_dim;
    int      rot_dim;        /* elements [rot_dim, head_dim) pass through */
    int      n_axes;
    int      pairing;
    uint64_t phase[SP_MAX_HEAD_DIM / 2];  /* a step of one position, as a fraction of a turn times
                                             2^64: the angle is the low 64 bits of position * phase,
                                             exact to 2^-53 of a turn for each step at any position */
    uint8_t  axis[SP_MAX_HEAD_DIM / 2];   /* the axis whose position turns the pair */
} sp_rope_axes_t;

/* head_dim: a multiple of 8 up to SP_MAX_HEAD_DIM.  rot_dim: a multiple of
 * 16 up to head_dim.  sections[n_axes]: pairs of each axis, >= 0, together
 * rot_dim/2.  freq_factors: NULL or rot_dim/2 finite divisors (not zero) of the
 * frequencies.  A frequency is the 32-bit float nearest to the formula's value,
 * as in the tables that models are trained with.  Host only. */
int sp_rope_axes_init(sp_rope_axes_t *ra, int head_dim, int rot_dim, int pairing, int n_axes,
                      const int *sections, int flags, double theta, const float *freq_factors);

/* Rotates the queries and keys of n_tokens tokens in one launch:
 *   (x, y) -> (x cos a - y sin a, x sin a + y cos a),  a = pos[axis][token] * frequency
 * (inverse != 0: by -a, which is also the gradient's way back).
 *   d_pos   int32 [n_axes][n_tokens], any values
 *   d_q     [n_tokens][n_q_heads][head_dim], a token's rows q_stride elements
 *           after the last token's (0: n_q_heads * head_dim); d_k likewise.
 *           Either may be NULL with its outputs (that half is skipped).
 *   outputs the same shape with strides of their own; may be the inputs
 *           themselves (same pointer and stride), but not overlap them otherwise
 *   dtype   SP_DTYPE_F32 / _F16 / _BF16, of inputs and outputs; the rotation
 *           runs in 32 bits and is rounded once
 * Pointers and strides in bytes must be multiples of 16. */
int sp_cuda_rope_axes(const sp_rope_axes_t *ra, const int *d_pos, int n_tokens, const void *d_q,
                      long long q_stride, int n_q_heads, void *d_q_out, long long q_out_stride,
                      const void *d_k, long long k_stride, int n_k_heads, void *d_k_out,
                      long long k_out_stride, int dtype, int inverse, void *stream);

/* --------------------------------------------------------- the cache -- */

/* Code formats: value = code * scale of the block. */
#define SP_Q8_INT8 0   /* signed byte in [-127, 127] */
#define SP_Q8_E4M3 1   /* 8-bit float: sign, 4 exponent bits, 3 mantissa bits, largest 448 */

/* A block is block_tokens consecutive positions of one slot (one layer,
 * sequence and KV head); it has one scale, and with Q = 127 or 448
 *     scale = max|x| * (1 / Q)  held within [2^-40, 2^40]
 *     code  = x * (1 / scale) rounded to the nearest code, ties to even, saturated
 * in 32-bit floats.  Infinities do not count for the maximum and saturate; NaN
 * is stored as 0. */
typedef struct {
    sp_config_t   config;        /* head_dim, n_layers and n_heads_kv are used */
    int           format;        /* SP_Q8_* */
    int           block_tokens;  /* 16, 32, 64 or 128 */
    int           n_seqs;        /* sequences held */
    int           max_seq_len;   /* positions of a sequence, rounded up to a multiple of 128 */
    void         *d_k_cache;     /* start of the one allocation: [n_layers][n_seqs][n_heads_kv][max_seq_len][head_dim] codes */
    void         *d_v_cache;
    float        *d_k_scale;     /* [n_layers][n_seqs][n_heads_kv][max_seq_len / block_tokens] */
    float        *d_v_scale;
    void         *stream;        /* of the writes and reads */
    int           n_slots;       /* n_layers * n_seqs * n_heads_kv */
    int           device;
    int           sm_count;
    void         *d_attn_ws;     /* partial results of the attention's split rows */
    size_t        attn_ws_bytes;
    unsigned int *d_status;      /* device error word: bit 0 a batch entry was out of range and
                                    skipped, bit 1 a bounded wait inside a kernel ran out */
} sp_cuda_q8_cache_t;

/* The new tokens of one step, packed one sequence after another.  The arrays
 * are in device memory, so a step's graph can be replayed with other lengths.
 * Entry i is skipped, and bit 0 of the status word set, unless
 *     0 <= d_cu[i] <= d_cu[i+1] <= n_tokens, d_cu[i+1] - d_cu[i] <= max_new,
 *     0 <= d_kv_len[i] <= max_kv, 0 <= d_seq[i] < n_seqs of the cache.
 * No two entries share packed tokens.  Where d_cu descends (which sets bit 0) they
 * may, and a write may then leave blocks out that come after n_tokens' worth. */
typedef struct {
    int        n_seqs;     /* entries, any number >= 0 */
    int        n_tokens;   /* packed tokens of all entries */
    int        max_new;    /* at least the most new tokens of an entry */
    int        max_kv;     /* at least the largest d_kv_len, at most max_seq_len */
    const int *d_seq;      /* [n_seqs] sequence of each entry, all different; NULL: entry i is sequence i */
    const int *d_cu;       /* [n_seqs + 1] first packed token of each entry */
    const int *d_kv_len;   /* [n_seqs] positions held with the new tokens: entry i's new tokens are
                              the positions [d_kv_len[i] - new, d_kv_len[i]) */
} sp_cuda_q8_batch_t;

/* head_dim 64, 128 or 256.  Allocates the slabs (zeroed), the scales (zeroed)
 * and the attention's workspace, and synchronises the device. */
int  sp_cuda_q8_cache_init(sp_cuda_q8_cache_t *qc, const sp_config_t *cfg, int format,
                           int block_tokens, int n_seqs, int max_seq_len, void *stream);
void sp_cuda_q8_cache_free(sp_cuda_q8_cache_t *qc);

/* Quantises the batch's keys and values into layer `layer` in one launch.
 * d_k, d_v: [n_tokens][n_heads_kv][head_dim] of dtype, a token's rows
 * token_stride elements after the last token's (0: dense); NULL skips that
 * half.  Pointers and the stride in bytes must be multiples of 16.
 *
 * A write ends its sequence: positions before it keep their values, positions
 * after it are undefined until they are written.  Where it begins inside a
 * block, the block's scale can only grow (the larger of the old one and what
 * the new tokens ask for), and if it does, the codes before the write are
 * requantised: code * (old / new) rounded as above.  An entry whose
 * d_kv_len is less than its new tokens is out of range. */
int  sp_cuda_q8_write_kv_tokens(sp_cuda_q8_cache_t *qc, int layer, const sp_cuda_q8_batch_t *batch,
                                const void *d_k, const void *d_v, long long token_stride, int dtype);

/* Positions [start_pos, start_pos + n_tok) of one sequence's every head, which
 * 0 = K, 1 = V, to d_out [n_tok][n_heads_kv][head_dim] of dtype (16-byte
 * aligned): code * scale, rounded once. */
int  sp_cuda_q8_read_kv_tokens(const sp_cuda_q8_cache_t *qc, int which, int layer, int seq,
                               int start_pos, int n_tok, void *d_out, int dtype);

/* Attention of the batch's new tokens over layer `layer`:
 *     out[t][g] = sum_j p_j V[j],  p = softmax_j(logit_scale * q[t][g] . K[j])
 * over the cached positions j that token t sees: with p its own position
 * (kv_len - new + its place among its entry's new tokens),
 *     causal != 0:  j <= p, and j > p - window where window > 0
 *     causal == 0:  every j < kv_len (window must be 0)
 * A token that sees nothing has out = 0 and lse = -infinity.
 *   d_q, d_out  [n_tokens][n_q_heads][head_dim], SP_DTYPE_F16 or _BF16, with
 *               strides between tokens in elements (0: dense); 16-byte multiples
 *   n_q_heads   a multiple of n_heads_kv, at most 128 for each; query head g
 *               reads KV head g / (n_q_heads / n_heads_kv)
 *   d_lse       NULL or fp32 [n_tokens][n_q_heads]: log sum_j exp(logit_scale q.K[j]),
 *               to join this result with attention over other positions
 * Scores, the softmax's statistics and sums are held in 32 bits; queries are
 * rounded to fp16 after a power of two that brings a row's largest element to
 * [1, 2) (elements under 2^-14 of it lose bits), softmax weights to fp16,
 * relative to a running maximum, for the product with V.  Calls on one cache must not overlap on the GPU (they share
 * its workspace). */
int  sp_cuda_q8_attn(const sp_cuda_q8_cache_t *qc, int layer, const sp_cuda_q8_batch_t *batch,
                     const void *d_q, long long q_stride, int n_q_heads, int dtype,
                     float logit_scale, int causal, int window, void *d_out, long long out_stride,
                     float *d_lse, void *stream);

/* The cache's status word after the stream's work (synchronises `stream`);
 * clear != 0 resets it. */
int  sp_cuda_q8_status(const sp_cuda_q8_cache_t *qc, unsigned int *status_out, int clear, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* SHANNON_PRIME_Q8_H */
