/* C ABI of libtace_hip.so, second part: operators on rows of atoms -- table
 * lookup by token and its gradient, rows sorted by expert and back, dropout
 * from a counter-based generator, root-mean-square norm, the experts' products
 * -- and the step that trains them (AdamW over many tensors).  Conventions are tace_hip.h's (device
 * pointers of the caller, asynchronous on `stream`, 0 or a negative code and
 * tace_last_error()); this part has a version of its own.
 *
 * Row types: TACE_ROW_F32, _F64, _BF16, _F16.  Sums, weights and scales are
 * double for TACE_ROW_F64 and float otherwise ("the type's sums").  Indices
 * (`index_bytes` 4 or 8) outside their range are no error: their rows are
 * zero and take no gradient.  Calls that need 2^32 threads or more (one for
 * each move of up to 16 bytes) are refused.
 *
 * The same inputs at the same alignment give the same bits on every run.  The
 * order of a sum depends on the tokens or places as well as on the sizes, and
 * on the width of a move, which the channels and the rows' alignment set. */
#ifndef TACE_ROWS_H
#define TACE_ROWS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TACE_ROWS_ABI_VERSION 4
#define TACE_ROW_F32 0
#define TACE_ROW_F64 1
#define TACE_ROW_BF16 2
#define TACE_ROW_F16 3
#define TACE_ROW_MAX_BLOCKS 8

int tace_rows_abi_version(void);

/* out [n, channels]: row i is scale * table[tokens[i]] (table [vocab,
 * channels]), zeros for a token outside [0, vocab). */
int tace_embed_fwd(int type, int index_bytes, const void* table, const void* tokens, int64_t n, int64_t vocab,
                   int32_t channels, double scale, void* out, void* stream);

/* grad [vocab, channels]: row v is scale * the sum of g's rows (g [n,
 * channels]) whose token is v, zeros without any.  order [n] and rowptr
 * [vocab + 1] are tace_route_group's of the tokens; NULL where
 * tace_embed_grad_grouped is 0 (few rows or tokens, always for n = 0).  work:
 * tace_embed_grad_work bytes (16-byte aligned) of the same choice, grouped or
 * not; NULL where that is 0. */
int tace_embed_grad_grouped(int64_t n, int64_t vocab);
int64_t tace_embed_grad_work(int type, int64_t n, int64_t vocab, int32_t channels, int grouped);
int tace_embed_grad(int type, int index_bytes, const void* g, const void* tokens, const int32_t* order,
                    const int32_t* rowptr, int64_t n, int64_t vocab, int32_t channels, double scale, void* grad,
                    void* work, int64_t work_bytes, void* stream);

/* Positions 0 .. n-1 grouped by key, as tace_group_keys orders them (order
 * [n], rowptr [n_keys + 1]; positions with a key outside [0, n_keys) last), and
 * place [n] (may be NULL), place[order[r]] = r.  Key i is keys[i * stride], of
 * index_bytes 4 or 8.  work: tace_route_group_work int32.
 *
 * Tokens sorted by expert: slot s = t k + j is choice j of token t, its key the
 * expert; n = tokens k.  rows_end points to rowptr[experts]: rows from there on
 * belong to dropped slots.  A place outside [0, n) is taken for n - 1.  Rows
 * are `blocks` blocks of widths[b] elements (host array); a batch of R rows
 * holds block after block, each [R, widths[b]] (blocks = 1: ordinary rows). */
int64_t tace_route_group_work(int64_t n, int64_t n_keys);
int tace_route_group(int index_bytes, const void* keys, int64_t stride, int64_t n, int64_t n_keys, int32_t* rowptr,
                     int32_t* order, int32_t* place, int32_t* work, void* stream);
/* out row place[s] = weights[s] x row t(s) (weights NULL: 1), zeros where s is dropped */
int tace_route_dispatch(int type, const void* x, const void* weights, const int32_t* place, const int32_t* rows_end,
                        int64_t tokens, int32_t k, int32_t blocks, const int64_t* widths, void* out, void* stream);
/* out row t = sum over its kept slots of weights[s] y row place[s] */
int tace_route_combine(int type, const void* y, const void* weights, const int32_t* place, const int32_t* rows_end,
                       int64_t tokens, int32_t k, int32_t blocks, const int64_t* widths, void* out, void* stream);
/* dots[s] = <x row t(s), y row place[s]>, 0 where s is dropped; g_y (NULL: not
 * wanted): as tace_route_dispatch of x by weights, in the same pass */
int tace_route_dots(int type, const void* x, const void* y, const void* weights, const int32_t* place,
                    const int32_t* rows_end, int64_t tokens, int32_t k, int32_t blocks, const int64_t* widths,
                    void* g_y, void* dots, void* stream);

/* Dropout.  x: `blocks` blocks [rows, comps[b], channels]; one draw for each
 * (row, block, channel), shared by the comps[b] components: draw i = (row
 * blocks + b) channels + c is half i % 2 (low first) of word (i % 8) / 2 of
 * Philox-4x32 with 10 rounds on counter (i / 8, site, offset low, offset high)
 * under key (seed low, seed high).  out = draw >= threshold ? x 65536 / (65536 -
 * threshold) : 0, plus residual where given.  state: device int64 [2] (seed,
 * offset), or NULL for the two arguments.  threshold 0 .. 65536. */
int tace_dropout(int type, const void* x, const void* residual, const int64_t* state, int64_t seed, int64_t offset,
                 uint32_t site, int32_t threshold, int64_t rows, int32_t channels, int32_t blocks,
                 const int32_t* comps, void* out, void* stream);

/* Root-mean-square norm.  x: `blocks` blocks [rows, comps[b], channels], one
 * after the other (plain rows: one block of one component, channels = the
 * row).  For each (row, block), n = comps[b] channels elements:
 * h = x + residual (rounded; without a residual h is x and must be NULL),
 * q = 1 / sqrt(sum h^2 / n + eps), y = h q weight[b][channel].  weight [blocks,
 * channels] has the rows' type, or its sums' where weight_wide.  inv [rows,
 * blocks] (the type's sums, may be NULL) receives q.  scales (float [rows,
 * blocks], NULL: y has the rows' type): y receives e4m3 codes, y = code *
 * scale, scale = max |y| / 448; a row with a NaN has scale NaN, one below 2^-100
 * is zeros under scale 0.
 *
 * Backward: dh = the gradient of h (and so of x and of residual) given gy and gh
 * (NULL: none); dw [blocks, channels] (NULL: not wanted) has weight's type.
 * work: tace_rms_norm_bwd_work bytes, 16-byte aligned (may be NULL without dw). */
int tace_rms_norm_fwd(int type, const void* x, const void* residual, const void* weight, int weight_wide, int64_t rows,
                      int32_t channels, int32_t blocks, const int32_t* comps, double eps, void* h, void* y,
                      float* scales, void* inv, void* stream);
int64_t tace_rms_norm_bwd_work(int type, int64_t rows, int32_t channels, int32_t blocks, const int32_t* comps);
int tace_rms_norm_bwd(int type, const void* gy, const void* gh, const void* h, const void* weight, int weight_wide,
                      const void* inv, int64_t rows, int32_t channels, int32_t blocks, const int32_t* comps, void* dh,
                      void* dw, void* work, int64_t work_bytes, void* stream);

/* The experts' products.  Rows sorted by expert as tace_route_group's (rowptr
 * [experts + 1], rowptr[0] taken for 0; rows from rowptr[experts] on are dropped;
 * entries that fall or leave the rows give other groups, with reads and writes
 * inside the rows all the same) in `blocks` blocks of
 * comps[b] components: a batch is block after block, each [rows, comps[b], K].
 * weight [experts, blocks, K, N].
 * tace_expert_linear: out [.., N] = scale x weight[expert][block], or (transposed;
 * x [.., N]) out [.., K] = scale x weight^T; zeros for dropped rows.
 * tace_expert_linear_grad: dw = scale x^T g of each expert's rows, zeros without
 * any; work: tace_expert_linear_grad_work bytes, 16-byte aligned, NULL where 0.
 * Products are summed in float (double for TACE_ROW_F64), float32's as six
 * products of three bfloat16 terms each.
 * tace_expert_linear_e4m3: out [rows, N] (TACE_ROW_F32, _BF16 or _F16) = x_scale
 * w_scale[expert] (x codes, w codes), x codes [.., K], weight codes [experts, N,
 * K] (both 16-byte aligned, K a multiple of 16), w_scale [experts, N].  order
 * (tace_route_group's): sorted row r is x's row order[r] / choices, x [rows /
 * choices, K]; NULL: x [rows, K] is sorted. */
int tace_expert_linear(int type, int transposed, const void* x, const void* weight, const int32_t* rowptr, int64_t rows,
                       int32_t experts, int32_t blocks, const int32_t* comps, int32_t K, int32_t N, double scale,
                       void* out, void* stream);
int64_t tace_expert_linear_grad_work(int type, int64_t rows, int32_t experts, int32_t blocks, const int32_t* comps,
                                     int32_t K, int32_t N);
int tace_expert_linear_grad(int type, const void* x, const void* g, const int32_t* rowptr, int64_t rows, int32_t experts,
                            int32_t blocks, const int32_t* comps, int32_t K, int32_t N, double scale, void* dw, void* work,
                            int64_t work_bytes, void* stream);
int tace_expert_linear_e4m3(int out_type, const void* x, const float* x_scale, const int32_t* order, int32_t choices,
                            const void* weight, const float* w_scale, const int32_t* rowptr, int64_t rows,
                            int32_t experts, int32_t K, int32_t N, void* out, void* stream);

/* AdamW.  tensors: host array; p, g [n] of the row type, m, s [n] the states:
 * averages of g and g^2 in the type's sums, or (`eight`) of g and the root of the
 * average of g^2 as e4m3 codes with scales float [ceil(n / 256), 2]; master
 * (weights of 16 bits; may be NULL) [n] float, which p is rounded from.
 * counter: device int64 [2], the steps done and zero; the step counts itself.
 * lr_at (may be NULL): device learning rate, float or (lr_wide) double, used
 * instead of lr.  norm (may be NULL): tace_grad_norm's of all gradients, which are
 * multiplied by min(1, max_norm / norm); where it is infinite or NaN nothing
 * changes.  Draws of the codes: a function of (seed; position / 4, index in
 * `tensors`, step).
 *
 * tace_grad_norm: norm (double for TACE_ROW_F64, else float) = the 2-norm of all
 * g.  ticket: a device int64 that is zero before and after (counter + 1 will
 * do).  work: tace_grad_norm_work bytes, 8-byte aligned. */
#define TACE_ADAM_BLOCK 256
typedef struct {
  void* p;
  const void* g;
  void* m;
  void* s;
  void* master;
  void* scales;
  int64_t n;
} tace_adam_tensor;
int64_t tace_grad_norm_work(const tace_adam_tensor* tensors, int64_t count);
int tace_grad_norm(int type, const tace_adam_tensor* tensors, int64_t count, int64_t* ticket, void* norm, void* work,
                   int64_t work_bytes, void* stream);
int tace_adamw(int type, int eight, const tace_adam_tensor* tensors, int64_t count, int64_t* counter, double lr,
               const void* lr_at, int lr_wide, double beta1, double beta2, double eps, double decay, const void* norm,
               double max_norm, uint64_t seed, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TACE_ROWS_H */
