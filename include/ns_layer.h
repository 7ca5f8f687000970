/* ns_layer.h: what a hybrid model's layer does beside attention, for one token and for prompts - the state-space mixer
 * (short causal convolution and selective scan), the norms around a block, and products with 4-bit weights. nemotron-h's
 * engine runs such layers between its attention layers (ns_nh_*: ns_attn.h); none of these has a counterpart in the
 * reference's C ABI. All calls are queued on the ns_gpu's compute stream, return 0 or -1 (+ ns_last_error()), allocate
 * nothing, record into a graph (kernel launches only) and give the same bits every time.
 *
 * Row types qt: 0 float32, 1 half, 2 bfloat16. Sums, norms, states and the convolution are float32. Strides are in
 * elements of their rows' type, at least a row long; rows may start at any element (they are read in wide pieces wherever
 * they start). Outputs overlap no input except where a call says that they may. */
#ifndef NS_LAYER_H
#define NS_LAYER_H
#include <stdint.h>
#include "ns.h"
#ifdef __cplusplus
extern "C" {
#endif

/* ---- the state-space mixer. H heads of P features, G groups of H / G heads that share B and C of N features;
 * a projected row is x [H][P] | B [G][N] | C [G][N], `chan` = H P + 2 G N values, and a step size [H]. For the row at
 * position p, with u(p) the raw row (zeros in front of position 0):
 *   c = silu(sum over k < K of cw[:][k] u(p - K + 1 + k) + cb)                      -> x, B, C
 *   dt = softplus(step + dtb), held to dt_lo .. dt_hi
 *   h = exp(dt a) h + dt x (outer) B[group],  y = h C[group] + d x                  a head
 * cw [chan][K], cb [chan] or null, a, dtb, d [H] (dtb, d or null), all float32. K 1 to 4, N up to 256, H a multiple of G,
 * H and P up to 65536, chan up to 2^24. dt_lo and dt_hi: 0 and infinity where the model has no limits.
 * conv: a ring of `cap` raw rows [cap][chan] float32, the row of position p in slot p % cap; the K - 1 rows in front of a
 * call's first have to be there (none in front of position 0 is read: a new sequence needs no clearing). K 1: may be null.
 * State: [H][P][N] float32; h0 is read and h1 written, and they may be the same (h0 null: zeros). */

/* T rows of one sequence at positions p0 .. p0 + T - 1: y [T] rows of H P, h1, and the last min(T, K - 1) raw rows into
 * the ring (cap >= K - 1). Rows up to 2^23 values apart (xs). scratch: ns_ssm_prompt_scratch(..) floats, 16-byte aligned:
 * it grows with T up to 8192 rows (0: sizes that the call does not take). Up to 16 rows, where the ring holds K - 1 + T, run as
 * ns_ssm_step's do; else in blocks of 64 rows whose matrix products keep 22 bits of each operand (half rows too; of bfloat16
 * rows those that reach y alone 11) and nothing below 2^-38 of the largest value of a column of x or of the state, of a block's B
 * or C, or of a row's products of B and C with steps and decays; x enters the state times its row's step, the largest step with the
 * column's largest x. Exponents of decays are sums of the steps between two rows alone: a large step takes no bits of others'. Finite
 * values of a block whose largest ones' products pass float32's range may leave rows that do not hold them not finite. A value that is
 * not finite reaches what the recurrence takes it to, rows in front of it never. */
int64_t ns_ssm_prompt_scratch(int64_t T, int64_t H, int64_t P, int64_t N, int64_t G, int64_t K);
int ns_ssm_prompt(ns_gpu* g, int qt, const void* xbc, int64_t xs, const void* dt, int64_t dts, const float* cw, const float* cb, const float* a,
                  const float* dtb, const float* d, float dt_lo, float dt_hi, float* conv, int64_t cap, int64_t p0, int64_t T, int64_t H,
                  int64_t P, int64_t N, int64_t G, int64_t K, const float* h0, float* h1, void* y, int64_t ys, float* scratch);

/* R rows (up to 4096) of up to R sequences, one launch: conv [nslots][cap][chan], h0 / h1 [nslots][H][P][N]. Row r belongs
 * to slot slots[r] (slots null: to slot r, R <= nslots); a row whose slot is not 0 .. nslots - 1 is passed over, its y left
 * as it was. The rows of one slot are successive tokens of its sequence, in the rows' order; its first is at position
 * pos[r] (pos null: p0). Every row goes into its slot's ring, so a sequence can be taken back to any row of the call whose
 * state the caller kept (h0 and h1 apart). A slot takes up to cap - K + 1 rows a call (cap >= K): the ring holds the rows
 * in front of them at the same time; rows of a slot beyond that are passed over too, and all of a slot whose first is at a
 * negative position. Slots that have no row: nothing of theirs is written. A row's results have the same bits in a call of its own and among others. */
int ns_ssm_step(ns_gpu* g, int qt, const void* xbc, int64_t xs, const void* dt, int64_t dts, const float* cw, const float* cb, const float* a,
                const float* dtb, const float* d, float dt_lo, float dt_hi, float* conv, int64_t cap, int64_t p0, const int32_t* pos,
                const int32_t* slots, int64_t nslots, int64_t R, int64_t H, int64_t P, int64_t N, int64_t G, int64_t K, const float* h0,
                float* h1, void* y, int64_t ys);

/* ---- norms. rms(v) = v / sqrt(mean(v^2) + eps). A call's groups (rows) are a launch's: fewer than 2^32 threads, 64 of them a
 * group of up to 64 pieces of 16 bytes (rounded up to 4 groups), 64 for each 64 pieces, 1024 at most, a longer one. */

/* The norm behind the scan, over each of `groups` equal parts of a row of D: order 0 out = rms(y silu(z)) w, order 1
 * out = rms(y) w silu(z); w [D] float32 or null (ones). Rows y, z, out of type qt; out may be y or z. */
int ns_norm_gated(ns_gpu* g, int qt, const void* y, int64_t ys, const void* z, int64_t zs, const float* w, void* out, int64_t os, int64_t T,
                  int64_t D, int64_t groups, float eps, int order);

/* A block's output into the residual stream and the norm in front of the next block: v = x, or rms(x) post with a norm
 * behind the block; s = h + scale gate v; h1 = s; out = rms(s) pre. x and out rows of type qt, h and h1 of type rt (0, or
 * qt); post, gate, pre [D] float32 or null (gate, pre: ones). x null: s = h (a model's first norm; post and gate null).
 * h1 or out null: not wanted. s is not rounded to rt in front of the norm. h1 may be h, out may be x. */
int ns_norm_residual(ns_gpu* g, int qt, int rt, const void* x, int64_t xs, const void* h, int64_t hs, void* h1, int64_t h1s, void* out, int64_t os,
                     int64_t T, int64_t D, float eps, float scale, const float* post, const float* gate, const float* pre);

/* ---- 4-bit weights. w[m][k] = (q - 8) s, q 0..15, a half scale s for each `group` (32, 64 or 128) of a row's values.
 * Held in tiles of 16 rows x 128 values, [ceil(M / 16)][ceil(K / 128)], each 1024 bytes of nibbles and 16 (128 / group)
 * scales: value (m, k) of a tile is a nibble of byte 16 (m + 16 (k / 8 % 4)) + 4 (k / 32) + (e % 2) 2 + e / 4, e = k % 8:
 * the low one where e / 2 is even, else the high one; its scale is entry (m / 4) 4 (128 / group) + (k / group) 4 + m % 4.
 * Values past M or K: q 8, scale 0. ns_q4_bytes: a matrix's bytes (16-byte aligned memory). */
int64_t ns_q4_bytes(int64_t M, int64_t K, int64_t group);
/* Lays out M rows of K values: form 0 float32 rows ss values apart, each group rounded by the q4_0 rule (s = the value of
 * the largest magnitude, the first of a tie, / -8; q = min(15, (int) (v / s + 8.5))); form 1 q4_0 blocks as model files
 * hold them (18 bytes: a half scale, then 16 bytes that pair value j with j + 16; group 32, K a multiple of 32), rows ss
 * bytes apart. Fewer than 2^32 groups (rows rounded up to 16, values to 128) a call. */
int ns_q4_pack(ns_gpu* g, int form, const void* src, int64_t ss, int64_t M, int64_t K, int64_t group, void* w);
/* y [T][M] = x [T][K] . w^T, 1 to 16 rows (a token, or a verify pass's rows), rows of type qt. The weights are exact in
 * the products; float32 rows enter as two halfs (22 bits), half rows as they are, bfloat16 rows too but for
 * what lies below 2^-29 of the largest of a row's 128 values. M up to 2^27 - 16, K up to 2^22. A row has the
 * same bits alone and among others. Rows that take more than 64 KiB as operands (16 half rows or 8 float32 rows of more
 * than 1920 values) are laid out in the library's own scratch by a launch in front, in order with the handle's other calls. */
int ns_q4_product(ns_gpu* g, int qt, const void* x, int64_t xs, const void* w, int64_t group, void* y, int64_t ys, int64_t T, int64_t M, int64_t K);

#ifdef __cplusplus
}
#endif
#endif
