/*
 * nabla_ops.h -- C ABI of the operators beside the optimizer step: the embedding lookup, its
 * gradient, and dropout from a counter-based generator.
 *
 * They feed the tensors that nabla_optim.h's lists describe: the embedding matrix is the largest
 * parameter of a language model, its gradient is the one that is not a matrix product, and dropout
 * is an element-wise pass like the Backend primitives.  The conventions are nabla_optim.h's: every
 * function returns an nbo_status and leaves a message for nbo_last_error(), nothing throws, all
 * work is enqueued on the library's stream (nbo_set_stream) on device 0 in call order, and what
 * returns nothing to the host does not synchronise.  The operators themselves allocate nothing and
 * may be captured into a HIP graph; their handles are created beforehand, and they and the tensors
 * stay for as long as the graph is replayed.
 */
#ifndef NABLA_OPS_H
#define NABLA_OPS_H

#include "nabla_optim.h"

#ifdef __cplusplus
extern "C" {
#endif

#pragma GCC visibility push(default)

/* A matrix in device memory: element (r, c) at data + (r * stride + c) elements of `dtype`.
 * Elements of a row are adjacent, stride >= cols (anything where there is at most one row), and the
 * address is a multiple of the element size.  It is taken as it is at the time of the call; like a
 * list's addresses it is checked against the allocation behind it (NBO_ERR_ARG; NBO_CHECK_POINTERS=0
 * in the environment skips that).  At most 2^31 - 2 rows and 2^27 columns (NBO_ERR_TOO_LARGE). */
typedef struct nbo_matrix {
    void *data;
    uint64_t rows, cols, stride;
    int32_t dtype; /* nbo_dtype */
    int32_t reserved;
} nbo_matrix;

/* Token ids: `n` integers at a device address, adjacent. */
typedef enum nbo_id_type { NBO_ID_I32 = 0, NBO_ID_I64 = 1 } nbo_id_type;
typedef struct nbo_ids {
    const void *data;
    uint64_t n;
    int32_t type; /* nbo_id_type */
    int32_t reserved;
} nbo_ids;

/* ---- embedding ------------------------------------------------------------------------- */

/* out[t] = add[t] + scale * table[ids[t]], t = 0 .. n - 1; `add` may be null (zeros).  An id that is
 * negative or not below table->rows (padding) stands for a row of zeros.  Computed in f32 (f64
 * tables: f64) and rounded once, to out's type: the table's type, or bf16 / f16 over an f32 table.
 * `add` has out's type and may be the very same matrix; other overlaps are NBO_ERR_ARG.  out and
 * add: ids->n rows, table->cols columns (NBO_ERR_SHAPE).  Asynchronous. */
int nbo_embedding(const nbo_matrix *table, const nbo_ids *ids, const nbo_matrix *add, double scale,
                  const nbo_matrix *out);

/* Scratch of nbo_embedding_grad for up to max_ids ids and max_cols columns: the ids ordered by rows
 * and partial sums of rows that many tokens name.  Nothing in it outlives a call, but two calls
 * that run at the same time (two captured graphs on two streams) need one each. */
typedef struct nbo_embedding_ws nbo_embedding_ws;
int nbo_embedding_ws_create(uint64_t max_ids, uint64_t max_cols, nbo_embedding_ws **out);
int nbo_embedding_ws_destroy(nbo_embedding_ws *ws);

/* The gradient of nbo_embedding with respect to the table:
 *   grad[v] = (accumulate ? grad[v] : 0) + scale * sum of grad_out[t] over the t with ids[t] == v
 * With accumulate == 0 every row is written, zeros where no id names it; otherwise the rows no id
 * names are not touched.  What rows of grad_out hold whose id is outside the table does not matter.
 * Sums are f32 (f64 tensors: f64), over the tokens in a fixed order -- the same bits on every run --
 * and rounded once, to grad's type: grad_out's, or f32 over bf16 / f16.  (With respect to `add` the
 * gradient is grad_out itself.)  grad may not overlap grad_out or the ids.  Asynchronous. */
int nbo_embedding_grad(const nbo_matrix *grad_out, const nbo_ids *ids, double scale, int accumulate,
                       const nbo_matrix *grad, nbo_embedding_ws *ws);

/* ---- dropout --------------------------------------------------------------------------- */

/* The generator's state, on the device: a seed and a step.  Masks are a function of (seed, step,
 * site, element); nothing is stored.  The step is advanced once a micro-batch, after its backward
 * pass, so that forward and backward of one micro-batch see the same masks and the next one sees
 * others -- in a captured graph too, where the advance is a node. */
typedef struct nbo_rng nbo_rng;
int nbo_rng_create(uint64_t seed, uint64_t step, nbo_rng **out);
int nbo_rng_destroy(nbo_rng *rng);
int nbo_rng_state_get(nbo_rng *rng, uint64_t *seed, uint64_t *step); /* synchronous */
int nbo_rng_load_state(nbo_rng *rng, uint64_t seed, uint64_t step);
int nbo_rng_advance(nbo_rng *rng, uint64_t steps); /* step += steps (modulo 2^64); asynchronous */

/* out[e] = residual[e] + (kept(e) ? x[e] * 65536 / (65536 - thr) : 0); `residual` may be null.
 * thr = floor(65536 p + 1/2): the drop rate is p to the nearest 2^-16, and the factor belongs to the
 * rate that is applied, so the mean is exact.  0 <= p <= 1 (NBO_ERR_ARG); p = 1 drops everything.
 * Element e = row * cols + col is dropped if its 16 bits of Philox4x32-10 are below thr: key = seed;
 * counter = (e / 8, site, step's low half, step's high half); the bits are half e % 2 (low first) of
 * word e % 8 / 2.  `site` tells the dropouts of one step apart (one number per place in the model).  A
 * dropped element is zero whatever x holds there (inf, NaN).  The gradient is the same call on the
 * gradient, without residual, at the same seed, step and site.  Computed in f32 (f64: f64), rounded
 * once.  x, residual and out have one shape and type; out may be x or residual itself, other overlaps
 * are NBO_ERR_ARG.  At most 2^35 elements.  Asynchronous. */
int nbo_dropout(const nbo_matrix *x, const nbo_matrix *residual, double p, nbo_rng *rng, uint32_t site,
                const nbo_matrix *out);

#pragma GCC visibility pop

#ifdef __cplusplus
}
#endif
#endif
