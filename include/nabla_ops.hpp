// nabla_ops.hpp -- C++ host side of nabla_ops.h: embedding lookup, its gradient, dropout.
// Header-only; link libnabla_optim.so.  Tensors are nabla_optim.hpp's (dense rows); errors are its
// exceptions: Panic for shapes that do not match, RuntimeError otherwise.
#ifndef NABLA_OPS_HPP
#define NABLA_OPS_HPP

#include <cstdint>

#include "nabla_ops.h"
#include "nabla_optim.hpp"

namespace nabla {
namespace ops {

using optim::Tensor;
using optim::check;

// `n` adjacent integers in device memory
struct Ids {
    const void *data = nullptr;
    uint64_t n = 0;
    int type = NBO_ID_I64;
};

inline nbo_matrix matrix(const Tensor &t) { return nbo_matrix{t.data, t.rows, t.cols, t.cols, t.dtype, 0}; }
inline nbo_ids ids_of(const Ids &i) { return nbo_ids{i.data, i.n, i.type, 0}; }

// out[t] = add[t] + scale * table[ids[t]]; without `add`, scale * table[ids[t]]
inline void embedding(const Tensor &table, const Ids &ids, const Tensor &out, double scale = 1.0, const Tensor *add = nullptr)
{
    const nbo_matrix t = matrix(table), o = matrix(out), a = add ? matrix(*add) : nbo_matrix{};
    const nbo_ids i = ids_of(ids);
    check(nbo_embedding(&t, &i, add ? &a : nullptr, scale, &o));
}

class EmbeddingWorkspace {
public:
    EmbeddingWorkspace(uint64_t max_ids, uint64_t max_cols) { check(nbo_embedding_ws_create(max_ids, max_cols, &h_)); }
    ~EmbeddingWorkspace() { (void)nbo_embedding_ws_destroy(h_); }
    EmbeddingWorkspace(const EmbeddingWorkspace &) = delete;
    EmbeddingWorkspace &operator=(const EmbeddingWorkspace &) = delete;
    nbo_embedding_ws *handle() const { return h_; }

private:
    nbo_embedding_ws *h_ = nullptr;
};

// grad[v] = (accumulate ? grad[v] : 0) + scale * sum of grad_out[t] over ids[t] == v
inline void embedding_grad(const Tensor &grad_out, const Ids &ids, const Tensor &grad, const EmbeddingWorkspace &ws,
                           double scale = 1.0, bool accumulate = false)
{
    const nbo_matrix d = matrix(grad_out), g = matrix(grad);
    const nbo_ids i = ids_of(ids);
    check(nbo_embedding_grad(&d, &i, scale, accumulate ? 1 : 0, &g, ws.handle()));
}

// The counter-based generator's state, on the device; advance() once a micro-batch.
class DropoutRng {
public:
    struct State {
        uint64_t seed, step;
    };
    explicit DropoutRng(uint64_t seed, uint64_t step = 0) { check(nbo_rng_create(seed, step, &h_)); }
    ~DropoutRng() { (void)nbo_rng_destroy(h_); }
    DropoutRng(const DropoutRng &) = delete;
    DropoutRng &operator=(const DropoutRng &) = delete;
    void advance(uint64_t steps = 1) { check(nbo_rng_advance(h_, steps)); }
    State state() const
    {
        State s{};
        check(nbo_rng_state_get(h_, &s.seed, &s.step));
        return s;
    }
    void load_state(const State &s) { check(nbo_rng_load_state(h_, s.seed, s.step)); }
    nbo_rng *handle() const { return h_; }

private:
    nbo_rng *h_ = nullptr;
};

// out = residual + (kept ? x / (1 - p) : 0)
inline void dropout(const Tensor &x, double p, const DropoutRng &rng, uint32_t site, const Tensor &out,
                    const Tensor *residual = nullptr)
{
    const nbo_matrix m = matrix(x), o = matrix(out), r = residual ? matrix(*residual) : nbo_matrix{};
    check(nbo_dropout(&m, residual ? &r : nullptr, p, rng.handle(), site, &o));
}
// its gradient with respect to x, at the same step and site
inline void dropout_grad(const Tensor &grad_out, double p, const DropoutRng &rng, uint32_t site, const Tensor &out)
{
    dropout(grad_out, p, rng, site, out);
}

} // namespace ops
} // namespace nabla
#endif
