// The C++ host side of the operators (include/nabla_ops.hpp) on the device: an input block forward and
// backward against the same sums on the host, in f64.  Exit code 0 = all passed.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../include/nabla_ops.hpp"

using namespace nabla::ops;

static int failures = 0;
#define EXPECT(cond)                                                        \
    do {                                                                    \
        if (!(cond)) {                                                      \
            std::printf("  FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            failures++;                                                     \
        }                                                                   \
    } while (0)

template <typename T> struct Dev {
    T *d = nullptr;
    size_t n;
    explicit Dev(const std::vector<T> &v) : n(v.size())
    {
        if (hipMalloc((void **)&d, n * sizeof(T)) != hipSuccess) std::abort();
        if (hipMemcpy(d, v.data(), n * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) std::abort();
    }
    ~Dev() { (void)hipFree(d); }
    std::vector<T> host() const
    {
        nabla::optim::sync();
        std::vector<T> v(n);
        if (hipMemcpy(v.data(), d, n * sizeof(T), hipMemcpyDeviceToHost) != hipSuccess) std::abort();
        return v;
    }
};

int main()
{
    const uint64_t rows = 50, cols = 24, n = 700;
    std::vector<double> table(rows * cols), dy(n * cols), grad(rows * cols, 0.25), out(n * cols, 9.0);
    std::vector<int64_t> ids(n);
    for (size_t i = 0; i < table.size(); i++) table[i] = std::sin(0.37 * (double)i);
    for (size_t i = 0; i < dy.size(); i++) dy[i] = std::cos(0.11 * (double)i);
    for (size_t t = 0; t < n; t++) ids[t] = t % 7 == 3 ? -1 : (int64_t)((t * t + 3 * t) % rows);
    Dev<double> dtable(table), ddy(dy), dgrad(grad), dout(out);
    Dev<int64_t> dids(ids);
    const Tensor T{dtable.d, rows, cols, NBO_DT_F64}, DY{ddy.d, n, cols, NBO_DT_F64}, G{dgrad.d, rows, cols, NBO_DT_F64},
        O{dout.d, n, cols, NBO_DT_F64};
    const Ids I{dids.d, n, NBO_ID_I64};

    embedding(T, I, O, 3.0);
    std::vector<double> got = dout.host();
    for (size_t t = 0; t < n; t++)
        for (size_t c = 0; c < cols; c++)
            EXPECT(got[t * cols + c] == (ids[t] < 0 ? 0.0 : 3.0 * table[(size_t)ids[t] * cols + c]));

    EmbeddingWorkspace ws(n, cols);
    embedding_grad(DY, I, G, ws, 0.5, true);
    std::vector<double> sum(rows * cols, 0.0), size(rows * cols, 0.0);
    for (size_t t = 0; t < n; t++)
        if (ids[t] >= 0)
            for (size_t c = 0; c < cols; c++) {
                sum[(size_t)ids[t] * cols + c] += dy[t * cols + c];
                size[(size_t)ids[t] * cols + c] += std::fabs(dy[t * cols + c]);
            }
    got = dgrad.host();
    for (size_t i = 0; i < sum.size(); i++) // two sums of at most 700 terms in different orders
        EXPECT(std::fabs(got[i] - (0.25 + 0.5 * sum[i])) <= (2 * 700 * size[i] + 4) * std::ldexp(1.0, -53));

    DropoutRng rng(123, 4);
    dropout(DY, 0.25, rng, 1, O);
    const std::vector<double> once = dout.host();
    size_t kept = 0;
    for (size_t i = 0; i < once.size(); i++) {
        EXPECT(once[i] == 0.0 || once[i] == dy[i] * (65536.0 / (65536.0 - 16384.0)));
        kept += once[i] != 0.0;
    }
    // 16800 draws at 0.75: a deviation of sqrt(16800 * 0.75 * 0.25) = 56
    EXPECT(std::fabs((double)kept - 12600.0) < 5 * 56.2);
    dropout_grad(DY, 0.25, rng, 1, O);
    EXPECT(dout.host() == once);
    rng.advance();
    EXPECT(rng.state().seed == 123 && rng.state().step == 5);
    dropout(DY, 0.25, rng, 1, O);
    EXPECT(dout.host() != once);
    rng.load_state({123, 4});
    dropout(DY, 0.25, rng, 1, O, &DY);
    got = dout.host();
    for (size_t i = 0; i < got.size(); i++) EXPECT(got[i] == dy[i] + once[i]);

    bool thrown = false;
    try {
        embedding(T, I, Tensor{dout.d, n, cols - 1, NBO_DT_F64});
    } catch (const nabla::optim::Panic &) {
        thrown = true;
    }
    EXPECT(thrown);
    thrown = false;
    try { // one element more than the allocation holds
        embedding(T, Ids{dids.d, n + 4096, NBO_ID_I64}, Tensor{dout.d, n + 4096, cols, NBO_DT_F64});
    } catch (const nabla::optim::RuntimeError &) {
        thrown = true;
    }
    EXPECT(thrown);
    std::printf("%d failure(s)\n", failures);
    return failures ? 1 : 0;
}
