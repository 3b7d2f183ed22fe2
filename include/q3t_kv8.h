/*
 * q3t_kv8.h -- C ABI of the operators of an 8-bit attention cache on MI355X
 * (gfx950): rotary positions, rows quantised into the cache, attention over
 * it, eviction by accumulated attention weight, and values read back.
 *
 * The talker runs on them when its cache type is Q3T_TYPE_I8
 * (q3t_dev_kv_set_type); a program that keeps caches of its own (more
 * streams, other head layouts) calls them on its own device memory.  The
 * reference has no counterpart: its cache is F16 and ends at n_ctx
 * (src/tts_transformer.cpp:731-783).
 *
 * Calls only launch kernels: every pointer is device memory of HIP device
 * `device` unless its comment says otherwise, `stream` is a hipStream_t of
 * that device (NULL: its default stream), nothing is allocated, copied to the
 * host or waited for, and a call may be captured into a hipGraph.  They hold
 * no state: calls on different streams or host threads may overlap as long as
 * they do not write the same memory (workspaces included).  The current HIP
 * device is the same after a call as before.
 * Status codes: 0 = ok, negative = refused or failed before anything was
 * launched (message from q3t_kv8_last_error).  Arguments on the host are
 * checked by the call.  Lengths and positions on the device cannot be: what
 * they may hold, and what a kernel does with other values, stands beside them;
 * no value makes a kernel leave the memory that the arguments describe.
 *
 * The cache of one layer: n_seq sequences of n_kv_head heads of n_slots
 * slots.  A slot of a head is a key and a value row of head_dim int8 codes;
 * 16 slots of a head (slots 16b .. 16b + 15) share one fp32 key scale and one
 * fp32 value scale, finite and not negative, and a code stands for
 * code * scale.  Slots are in the order of time; a slot's row was rotated for
 * its position before it was stored, so attention needs no positions and slots
 * may be evicted.
 */
#ifndef Q3T_KV8_H
#define Q3T_KV8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types (ggml ids, as in q3t_dev.h): 0 = F32, 1 = F16, 30 = BF16. */

#define Q3T_KV8_BLOCK 16  /* slots that share a scale */

typedef struct q3t_kv8 {
    int8_t * k, * v;          /* codes of sequence s, head h, slot t: k + s * seq + h * head + t * head_dim (bytes) */
    float * ks, * vs;         /* scales of block b: ks + s * scale_seq + h * scale_head + b (floats) */
    float * acc;              /* weight that slot t has drawn: acc + s * acc_seq + h * acc_head + t; NULL: not kept */
    int64_t seq, head;        /* multiples of 16, as k and v are */
    int64_t scale_seq, scale_head, acc_seq, acc_head;
    int32_t n_seq, n_kv_head; /* up to 65,535 and 4,096, 2^23 together */
    int32_t n_slots;          /* a multiple of 16, up to 2^29 */
    int32_t head_dim;         /* 64 or 128 */
} q3t_kv8;

/* Message of this host thread's last failed call ("" if none). */
const char * q3t_kv8_last_error(void);

/* ---------------------------------------------------------------- rotary */

/* Frequencies of rotary pairs i < rot_dim / 2, written to freq_out (HOST
 * memory, rot_dim / 2 doubles): theta^(-2 i / rot_dim), scaled for contexts
 * `factor` times the trained n_trained positions (factor 1: as trained):
 *   scaling 0  none (factor is not read)
 *   scaling 1  all divided by factor
 *   scaling 2  theta * factor^(rot_dim / (rot_dim - 2)) in place of theta
 *   scaling 3  those with more than 32 turns in n_trained positions as they
 *              are, those with less than one divided by factor, in between a
 *              mixture, linear in the logarithm of the turns. */
int q3t_kv8_rope_freqs(int32_t rot_dim, double theta, int32_t scaling, double factor, int32_t n_trained,
                       double * freq_out);

/* One tensor of rows: element d of head h of token t at
 * x + t * x_token + h * x_head + d (strides in elements). */
typedef struct q3t_kv8_rope_rows {
    const void * x; void * y;          /* y == x (same type and strides): in place; else no overlap */
    int64_t x_token, x_head, y_token, y_head;
    const float * gain;                /* [head_dim] of the RMS norm before the rotation; NULL: no norm */
    int32_t n_head;
    int32_t x_type, y_type;
} q3t_kv8_rope_rows;

/* Rotates the first rot_dim dims of every row of n (1 to 4) tensors by
 * their token's position: with z = x, or x / sqrt(mean(x^2) + eps) * gain,
 * the pair (z_i, z_{i + rot_dim / 2}), or (z_2i, z_{2i + 1}) where interleaved,
 * turns by pos * freq[i] and is multiplied by mscale; dims from rot_dim on are
 * z's.  Token t's position is pos[t] + pos0 (pos NULL: t + pos0).  Angles are
 * taken in 64 bits, the rest is 32-bit and rounded once.
 * head_dim: a multiple of 16 up to 256; rot_dim: even, 2 .. head_dim;
 * freq: [rot_dim / 2] (device); n_tokens: 0 to 2^26. */
int q3t_kv8_rope(int32_t device, const q3t_kv8_rope_rows * rows, int32_t n, int64_t n_tokens, int32_t head_dim,
                 int32_t rot_dim, int32_t interleaved, const int32_t * pos, int32_t pos0, const double * freq,
                 float mscale, float eps, void * stream);

/* ---------------------------------------------------------------- append */

/* Stores n_rows rows of each sequence (up to 2^26): row i of sequence s, head
 * h, at k + s * x_seq + i * x_row + h * x_head (strides in elements, of k and v
 * alike; type F32, F16 or BF16), goes to slot start[s] + start0 + i (start
 * NULL: start0 + i).  n_new[s] (NULL: n_rows; clamped to 0 .. n_rows): rows of
 * sequence s; the rest is padding that is not read.  A row whose slot is not in
 * 0 .. n_slots - 1 is not stored.
 * Per block of 16 slots and head: the scale becomes max(scale, a / 127) if the
 * block held slots before start, else a / 127, a the largest finite magnitude
 * of its new rows; codes before start move to the new scale where that grew,
 * rounded to nearest even; new codes are x / scale, rounded to nearest even,
 * at most 127 in size.  So a row stored in an earlier call may be rounded
 * again when its block's scale grows: at most half a step of the new scale
 * each time.  Infinities are stored as +-127, NaN as 0.  Codes of slots from
 * start + n_new on are left as they were, and not kept by a later append that
 * begins at or before them.
 * acc, where kept, is set to 0 for the new slots. */
int q3t_kv8_append(int32_t device, const q3t_kv8 * cache, const void * k, const void * v, int32_t type, int64_t x_seq,
                   int64_t x_row, int64_t x_head, int32_t n_rows, const int32_t * start, int32_t start0,
                   const int32_t * n_new, void * stream);

/* ------------------------------------------------------------- attention */

typedef struct q3t_kv8_attend_args {
    const void * q; void * out;       /* row i of sequence s, head h: q + s * q_seq + i * q_row + h * q_head (elements);
                                       * out overlaps nothing that is read */
    int64_t q_seq, q_row, q_head, o_seq, o_row, o_head;
    int32_t q_type;                   /* F16 or BF16 */
    int32_t o_type;                   /* F32, F16 or BF16 */
    int32_t n_rows, n_head;           /* n_rows up to 65,535; n_head: a multiple of n_kv_head, up to 32 times as many:
                                       * head h reads kv head h / (n_head / n_kv_head) */
    const int32_t * lens; int32_t len0;   /* sequence s has lens[s] + len0 slots, its new rows' among them (lens NULL:
                                           * len0); clamped to 0 .. max_len */
    const int32_t * n_new;            /* rows of each sequence (NULL: n_rows; clamped to 0 .. n_rows); out rows past
                                       * them are left as they were */
    int32_t max_len;                  /* the longest sequence the call is sized for; 0: n_slots */
    int32_t causal;                   /* 1: row i sees slots 0 .. len - n_new + i; 0: every row sees all len slots */
    float scale;                      /* of the scores, 1 / sqrt(head_dim) as a rule */
    int32_t weights;                  /* 1: acc of each slot grows by the probabilities it drew, summed over the rows
                                       * and the heads that read its kv head (in fp32, in a fixed order) */
} q3t_kv8_attend_args;

/* Bytes of workspace that q3t_kv8_attend needs for these arguments (0 is
 * possible); negative: refused.  Depends on the sizes alone, not on lens. */
int64_t q3t_kv8_attend_ws(const q3t_kv8 * cache, const q3t_kv8_attend_args * a);
/* Softmax attention of the rows of q over the cache.  A row that sees no
 * slot is 0; one that is not finite is NaN, and so are the weights of the slots
 * that it sees.  Scores, softmax and sums are fp32; probabilities enter the
 * value product as 11-bit numbers.  Codes of slots past a sequence's length are
 * not read into a result, whatever they hold.  ws: ws_bytes bytes, 16-byte
 * aligned, that no other work touches until this call's kernels are done (a
 * captured call keeps it for every replay). */
int q3t_kv8_attend(int32_t device, const q3t_kv8 * cache, const q3t_kv8_attend_args * a, void * ws, int64_t ws_bytes,
                   void * stream);

/* -------------------------------------------------------------- eviction */

/* Keeps min(len, n_keep) slots of every (sequence, head) of `from` and writes
 * them, in their order, to slots 0 .. of `to` (other memory, same sequences,
 * heads and head_dim; its n_slots at least n_keep): the first n_sink, the last
 * n_recent, and of the others those with the largest acc (equal ones: the
 * lowest slot first; NaN counts as -infinity).  n_sink + n_recent <= n_keep.
 * Both caches keep acc; it moves with its slot.  A block of `to` takes the
 * largest scale of its slots' old blocks, and codes move to it rounded to
 * nearest even.  lens, len0: as in q3t_kv8_attend, clamped to
 * 0 .. from->n_slots.  kept [n_seq][n_kv_head][n_keep] receives the kept slots'
 * old numbers, ascending, -1 behind them; len_out [n_seq] (NULL ok; lens
 * itself is fine) the new lengths.  Slots of `to` behind them are left as they
 * were. */
int q3t_kv8_evict(int32_t device, const q3t_kv8 * from, const q3t_kv8 * to, const int32_t * lens, int32_t len0,
                  int32_t n_keep, int32_t n_sink, int32_t n_recent, int32_t * kept, int32_t * len_out, void * stream);

/* ------------------------------------------------------------- read back */

/* The values of slots start[s] + start0 .. + n_rows - 1 (start NULL: start0 ..)
 * of every head, code * scale in fp32 and then rounded to `type`, as contiguous
 * [n_seq][n_rows][n_kv_head][head_dim] in k and v (16-byte aligned; either may
 * be NULL).  0 for slots outside the cache. */
int q3t_kv8_read(int32_t device, const q3t_kv8 * cache, const int32_t * start, int32_t start0, int32_t n_rows,
                 int32_t type, void * k, void * v, void * stream);

#ifdef __cplusplus
}
#endif
#endif
