/* ns_kv8.h: attention over a cache of 8-bit values in blocks of tokens, shared by any number of sequences, each block and key
 * head with one scale; and the eviction of its least attended tokens. None of these has a counterpart in the reference's C
 * ABI. All calls are queued on the ns_gpu's compute stream, return 0 or -1 (+ ns_last_error()), allocate nothing, record into a
 * graph (kernel launches only) and give the same bits every time; lengths, tables and starts are read on the device when the
 * call runs, so a recorded graph serves every token within the bounds that it was recorded with.
 *
 * The cache: pools kc, vc [blocks][Hkv][block][D] bytes and scales ksc, vsc [blocks][Hkv] float32, `block` 16, 32, 64 or 128
 * tokens, D 128 or 256. form 0: int8, codes -127 .. 127; 1: e4m3, magnitudes up to 448. A value is code x scale; a scale is a
 * power of two, 2^-24 .. 2^9 (int8) or 2^-15 .. 2^7 (e4m3), so a value is exactly a half. Pools 16-byte aligned. Nothing needs
 * clearing: a block's scale and codes count from its first token's store on.
 * Sequences: S of them, table [S][tmax] int32: token p of sequence s is row p % block of block table[s][p / block]. A token whose
 * entry is not a block of the pool, or lies past tmax, reads as a key and value of zeros, and nothing is written for it. Sequences
 * may share blocks that no call writes.
 * Rows of a call: sequence s has rows start[s] .. start[s + 1] - 1 of T (start [S + 1], ascending; null: row s alone, if s < T), the
 * first `most` of them; they are its tokens lens[s], lens[s] + 1, ... (lens [S] int32: the tokens in front of the call, up to 2^30). Rows
 * of no sequence, behind a sequence's first `most`, or of one whose lens is negative or larger: passed over, outputs left as they were.
 * Query heads: a multiple of the key heads, up to 4096 times as many.
 * Row types qt: 0 float32, 1 half, 2 bfloat16; strides in elements, at least a row long; rows may start at any element.
 * acc: float32 [blocks][Hkv][block], what each cached token has been given of the softmax weights, summed over rows and over the
 * query heads that share its key head. */
#ifndef NS_KV8_H
#define NS_KV8_H
#include <stdint.h>
#include "ns.h"
#ifdef __cplusplus
extern "C" {
#endif

/* Rows k, v (Hkv x D each) into their tokens' places. A block that a call writes from its first row on gets new scales: the
 * least power of two s with s M no less than the largest magnitude stored (M 127 or 448), held to the range above. In a block that
 * holds rows already, scales only grow, to what the new rows need, and the codes that were there are re-rounded to the new
 * unit: a value loses less than one step of the block's final scale, however often that grows. Codes are rounded to nearest even; NaN is
 * stored as 0, larger magnitudes as the largest. A block that the call writes belongs to one sequence. */
int ns_kv8_store(ns_gpu* g, int form, int qt, const void* k, int64_t ks, const void* v, int64_t vs, int64_t T, const int32_t* start, const int32_t* lens,
                 int64_t S, int64_t most, const int32_t* table, int64_t tmax, int64_t Hkv, int64_t D, int64_t block, int64_t blocks, void* kc,
                 void* vc, float* ksc, float* vsc);

/* Attention of a token, or a few (most 1 .. 16), of each of S sequences, whose keys are stored already: out [T][Hq D] =
 * softmax(scale q . k) v over the tokens up to the row's own, of the last `win` (win <= 0: of all); scale <= 0: 1 / sqrt(D). `longest`: no
 * token from that position on is read (a bound that the caller knows on every lens[s] + its rows; splits and scratch follow from it). S x most x Hq: under 2^31.
 * Half and bfloat16 rows enter the products exactly (values down to 2^-27 of a row and head's largest), float32 rows (of largest values from 2^-107 up) and the
 * softmax weights with 22 bits. A row that sees nothing: zeros. scratch:
 * ns_kv8_attend_scratch(..) floats, 16-byte aligned (0: may be null).
 * acc1 not null: acc1 = acc0 + the weights of this call's rows, for every token in front of lens[s] + its rows (acc0 null, and
 * tokens of this call: 0 + them; to tokens from `longest` on none are given); acc1 may be acc0. A block that is given weights belongs to one sequence of the call. */
int64_t ns_kv8_attend_scratch(int64_t S, int64_t most, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest, int acc);
int ns_kv8_attend(ns_gpu* g, int form, int qt, const void* q, int64_t qs, int64_t T, const int32_t* start, const int32_t* lens, int64_t S, int64_t most,
                  int64_t longest, const int32_t* table, int64_t tmax, int64_t Hq, int64_t Hkv, int64_t D, int64_t block, int64_t blocks, const void* kc,
                  const void* vc, const float* ksc, const float* vsc, int64_t win, float scale, void* out, const float* acc0, float* acc1, float* scratch);

/* A prompt's T rows, tokens p0 .. p0 + T - 1 of one sequence (table: its tmax entries), whose keys are stored already: the values are widened to half - exactly
 * - in the library's scratch and the pass runs as ns_attn_prompt_t's over a half cache (q and out 16-byte aligned, qs a multiple
 * of 16 bytes); up to 16 rows, and a pass whose values do not fit that scratch, as ns_kv8_attend's do. Rows and weights have ns_kv8_attend's bits and range whichever way
 * they go, but for half and bfloat16 rows' softmax weights in the pass: 11 bits, the same in a row's sum, off by no more than a half's rounding. */
int ns_kv8_prompt(ns_gpu* g, int form, int qt, const void* q, int64_t qs, int64_t T, const int32_t* table, int64_t tmax, int64_t p0, int64_t Hq, int64_t Hkv,
                  int64_t D, int64_t block, int64_t blocks, const void* kc, const void* vc, const float* ksc, const float* vsc, int64_t win, float scale,
                  void* out);

/* What T rows of one sequence, tokens p0 .. p0 + T - 1, give every token in front of p0 + T, without their outputs: acc1 as above (a prompt's last rows as
 * observers, or all of a prompt's passes one after another). */
int ns_kv8_weights(ns_gpu* g, int form, int qt, const void* q, int64_t qs, int64_t T, const int32_t* table, int64_t tmax, int64_t p0, int64_t Hq, int64_t Hkv,
                   int64_t D, int64_t block, int64_t blocks, const void* kc, const float* ksc, int64_t win, float scale, const float* acc0, float* acc1);

/* Shortens every sequence of more than `keep` tokens to `keep`, each key head for itself: its first `first` and last `last` tokens
 * (first + last <= keep) and of the others those of the largest acc (equal ones: the earliest; NaN and what is below 0 count as 0) keep their
 * order and move to tokens 0 .. keep - 1, acc with them. to null: within the sequence's own blocks, by way of the library's
 * scratch; else into the blocks of `to` [S][tmax], none of which may be a block that the call reads - sequences that stay as long as they are move too. A
 * block's scale becomes the largest of those its tokens come with, codes re-rounded as a store does. lens1 [S] = min(lens, keep)
 * (may be lens; sequences of negative lens: lens). No length is over `longest`, up to 2^30 (a longer sequence is passed over, its lens1 = lens); pools of
 * fewer than 2^32 rows, blocks x Hkv x block. */
int ns_kv8_evict(ns_gpu* g, int form, const int32_t* lens, int32_t* lens1, int64_t S, int64_t longest, int64_t keep, int64_t first, int64_t last,
                 const int32_t* table, const int32_t* to, int64_t tmax, int64_t Hkv, int64_t D, int64_t block, int64_t blocks, void* kc, void* vc,
                 float* ksc, float* vsc, float* acc);

#ifdef __cplusplus
}
#endif
#endif
