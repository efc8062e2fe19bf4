// The host side of the operators (nbo_ops.cpp) without a GPU, over a HIP runtime that notes what it is asked
// for.  One test to a run: `test_ops_host.bin NAME`; exit code 0 = passed.
#include "hip_stub.hpp"

#include <cstdio>

#include "../../include/nabla_ops.h"
#include "../../nabla_amd/csrc/nbo_ops_types.h"

static int failures = 0;
#define EXPECT(cond)                                                        \
    do {                                                                    \
        if (!(cond)) {                                                      \
            std::printf("  FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            failures++;                                                     \
        }                                                                   \
    } while (0)

namespace {
void *device(size_t bytes)
{
    void *p = nullptr;
    (void)hipMalloc(&p, bytes);
    return p;
}
nbo_matrix matrix(uint64_t rows, uint64_t cols, int dtype)
{
    return nbo_matrix{device(rows * cols * (dtype == NBO_DT_F64 ? 8 : dtype == NBO_DT_F32 ? 4 : 2)), rows, cols, cols, dtype, 0};
}
nbo_ids ids_of(uint64_t n) { return nbo_ids{device(n * 8), n, NBO_ID_I64, 0}; }

int lookup()
{
    const nbo_matrix table = matrix(9, 16, NBO_DT_F32), out = matrix(3, 16, NBO_DT_F32);
    const nbo_ids ids = ids_of(3);
    return nbo_embedding(&table, &ids, nullptr, 1.0, &out);
}

// A process that clears gradients (or steps an optimizer) loads one code object; the operators' comes
// with the first of them, inside a capture too.
void loads_the_operators_when_they_are_used()
{
    EXPECT(nbo_init() == NBO_OK);
    const uint64_t rows = 4, cols = 8;
    void *g = device(rows * cols * 4);
    nbo_list *list = nullptr;
    EXPECT(nbo_list_create(1, &rows, &cols, NBO_DT_F32, &g, &list) == NBO_OK);
    EXPECT(nbo_zero_grad(list) == NBO_OK);
    EXPECT(stub::modules.size() == 1);
    EXPECT(lookup() == NBO_OK);
    EXPECT(stub::modules.size() == 2 && stub::load_mode == hipStreamCaptureModeRelaxed &&
           stub::capture_mode == hipStreamCaptureModeGlobal);
    EXPECT(lookup() == NBO_OK);
    EXPECT(stub::modules.size() == 2);
}
void handles_load_the_operators()
{
    nbo_rng *rng = nullptr;
    EXPECT(nbo_rng_create(1, 2, &rng) == NBO_OK);
    EXPECT(stub::modules.size() == 2);
}
// An operators' code object that does not load takes nothing else with it, and is tried again.
void optimizers_do_without_the_operators()
{
    stub::fail_module = 1;
    EXPECT(nbo_init() == NBO_OK);
    EXPECT(lookup() == NBO_ERR_HIP + (int)hipErrorNoBinaryForGpu);
    EXPECT(stub::capture_mode == hipStreamCaptureModeGlobal);
    EXPECT(lookup() == NBO_OK);
}
// Which tensor it was, and where.
std::string at(const void *p)
{
    char text[32];
    std::snprintf(text, sizeof(text), " at %p: ", p);
    return text;
}
void addresses_are_named()
{
    EXPECT(nbo_init() == NBO_OK);
    const uint64_t rows[2] = {4, 4}, cols[2] = {8, 8};
    float host[32];
    void *good = device(128), *ptrs[2] = {good, host};
    nbo_list *list = nullptr;
    EXPECT(nbo_list_create(2, rows, cols, NBO_DT_F32, ptrs, &list) == NBO_ERR_ARG);
    EXPECT(nbo_last_error() == "tensor 1" + at(host) + "not memory the HIP runtime knows (a host pointer?)");
    ptrs[1] = (char *)good + 4;
    EXPECT(nbo_list_create(2, rows, cols, NBO_DT_F32, ptrs, &list) == NBO_ERR_ARG);
    EXPECT(nbo_last_error() == "tensor 1" + at(ptrs[1]) + "128 bytes do not fit the allocation (124 bytes from there to its end)");
    const nbo_matrix table = matrix(9, 16, NBO_DT_F32), out = matrix(3, 16, NBO_DT_F32);
    const nbo_ids ids = ids_of(3), beyond{ids.data, 4, NBO_ID_I64, 0}, on_host{host, 3, NBO_ID_I32, 0};
    nbo_matrix more = out;
    more.rows = 4;
    EXPECT(nbo_embedding(&table, &beyond, nullptr, 1.0, &more) == NBO_ERR_ARG);
    EXPECT(nbo_last_error() == "ids" + at(ids.data) + "32 bytes do not fit the allocation (24 bytes from there to its end)");
    EXPECT(nbo_embedding(&table, &on_host, nullptr, 1.0, &out) == NBO_ERR_ARG);
    EXPECT(nbo_last_error() == "ids" + at(host) + "not memory the HIP runtime knows (a host pointer?)");
}

// What runs for a gradient: `test_ops_host.bin plan IDS ROWS COLS TYPE GRAD_TYPE ACCUMULATE`, a launch to a line.
int plan(char **argv)
{
    auto number = [&](int k) { return std::strtoull(argv[k], nullptr, 10); };
    stub::args_bytes = [](const std::string &name) -> size_t {
        return name.compare(0, 14, "nbo_embed_sum_") == 0 || name.compare(0, 15, "nbo_embed_join_") == 0 ? sizeof(NboEmbedGradArgs)
               : name.compare(0, 10, "nbo_order_") == 0                                                   ? sizeof(NboOrderArgs)
                                                                                                          : 0;
    };
    const nbo_ids ids = ids_of(number(2));
    const nbo_matrix dy = matrix(ids.n, number(4), (int)number(5)), grad = matrix(number(3), number(4), (int)number(6));
    nbo_embedding_ws *ws = nullptr;
    EXPECT(nbo_embedding_ws_create(ids.n, grad.cols, &ws) == NBO_OK);
    stub::launches.clear();
    EXPECT(nbo_embedding_grad(&dy, &ids, 1.0, (int)number(7), &grad, ws) == NBO_OK);
    for (const stub::Launch &l : stub::launches) {
        std::printf("%s grid %u %u", l.name.c_str(), l.gx, l.gy);
        if (l.args.size() == sizeof(NboEmbedGradArgs)) {
            NboEmbedGradArgs a;
            std::memcpy((void *)&a, l.args.data(), sizeof(a));
            std::printf(" piece %u pieces %u lanes %u slabs %u edges %u", a.piece, a.pieces, a.lanes, a.slabs, a.edges);
        } else if (l.args.size() == sizeof(NboOrderArgs)) {
            NboOrderArgs a;
            std::memcpy((void *)&a, l.args.data(), sizeof(a));
            std::printf(" tiles %u digits %u range %u", a.tiles, a.digits, a.range);
        }
        std::printf("\n");
    }
    return failures;
}
} // namespace

int main(int argc, char **argv)
{
    const std::map<std::string, void (*)()> tests = {
        {"addresses_are_named", addresses_are_named},
        {"loads_the_operators_when_they_are_used", loads_the_operators_when_they_are_used},
        {"handles_load_the_operators", handles_load_the_operators},
        {"optimizers_do_without_the_operators", optimizers_do_without_the_operators},
    };
    if (argc < 2) {
        for (const auto &t : tests) std::printf("%s\n", t.first.c_str());
        return 0;
    }
    if (argc == 8 && argv[1] == std::string("plan")) return plan(argv);
    tests.at(argv[1])();
    std::printf("%d failure(s)\n", failures);
    return failures ? 1 : 0;
}
