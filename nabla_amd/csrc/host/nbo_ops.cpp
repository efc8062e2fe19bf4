// extern "C" entry points of include/nabla_ops.h: argument checks, the choice of kernels and their grids.
#include <algorithm>
#include <cmath>
#include <string>

#include "../../../include/nabla_ops.h"
#include "nbo_api_guard.hpp"
#include "nbo_host.hpp"

using namespace nbo;

namespace {

constexpr uint64_t MAX_ROWS = 0x7FFFFFFEull; // (one more is the key of ids outside the table)
constexpr uint64_t MAX_COLS = 1ull << 27;

uint64_t size_of(int dtype) { return dtype == NBO_DT_F64 ? 8 : is_half(dtype) ? 2 : 4; }

// The library's device for the time of a call: the caller's thread may have another one current.
class OnDevice {
public:
    explicit OnDevice(int device)
    {
        hip_check(hipGetDevice(&was_), "hipGetDevice");
        if (was_ != device) hip_check(hipSetDevice(device), "hipSetDevice");
        else was_ = -1;
    }
    ~OnDevice()
    {
        if (was_ >= 0) (void)hipSetDevice(was_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;

private:
    int was_ = -1;
};

// bytes from a matrix's first element to behind its last
uint64_t extent(const nbo_matrix &m)
{
    return m.rows && m.cols ? ((m.rows - 1) * m.stride + m.cols) * size_of(m.dtype) : 0;
}

// What can be said without the device: types, sizes, strides.
void check_form(const nbo_matrix *m, const char *what)
{
    if (!m) fail(NBO_ERR_ARG, std::string("null ") + what);
    if (m->dtype != NBO_DT_F32 && m->dtype != NBO_DT_BF16 && m->dtype != NBO_DT_F64 && m->dtype != NBO_DT_F16)
        fail(NBO_ERR_ARG, std::string(what) + ": unknown dtype");
    if (m->rows > MAX_ROWS || m->cols > MAX_COLS)
        fail(NBO_ERR_TOO_LARGE, std::string(what) + ": more than 2^31 - 2 rows or 2^27 columns");
    if (m->rows > 1 && m->stride < m->cols) fail(NBO_ERR_ARG, std::string(what) + ": rows overlap (stride < cols)");
    if (m->rows > 1 && m->stride > (UINT64_MAX >> 4) / m->rows)
        fail(NBO_ERR_TOO_LARGE, std::string(what) + ": the stride overflows 64 bits");
    if (m->rows && m->cols) {
        if (!m->data) fail(NBO_ERR_ARG, std::string("null device address for a non-empty ") + what);
        if ((uintptr_t)m->data % size_of(m->dtype))
            fail(NBO_ERR_ARG, std::string(what) + ": the address is not a multiple of the element size");
    }
}

void check_ids(const nbo_ids *ids)
{
    require(ids != nullptr, NBO_ERR_ARG, "null ids");
    require(ids->type == NBO_ID_I32 || ids->type == NBO_ID_I64, NBO_ERR_ARG, "ids: unknown integer type");
    require(ids->n <= MAX_ROWS, NBO_ERR_TOO_LARGE, "ids: more than 2^31 - 2");
    if (ids->n) {
        require(ids->data != nullptr, NBO_ERR_ARG, "null device address for non-empty ids");
        require((uintptr_t)ids->data % (ids->type == NBO_ID_I64 ? 8 : 4) == 0, NBO_ERR_ARG,
                "ids: the address is not a multiple of the element size");
    }
}

uint64_t id_bytes(const nbo_ids &ids) { return ids.n * (ids.type == NBO_ID_I64 ? 8 : 4); }

void check_shape(const nbo_matrix &m, uint64_t rows, uint64_t cols, const char *what)
{
    if (m.rows != rows || m.cols != cols)
        fail(NBO_ERR_SHAPE, std::string("nabla: ") + what + " (" + std::to_string(m.rows) + "x" + std::to_string(m.cols) +
                                ") vs (" + std::to_string(rows) + "x" + std::to_string(cols) + ") -- shapes must match");
}

// Whether two matrices have a byte in common.  Those of one row stride can lie side by side in one
// allocation (column slices); others count as overlapping when their address ranges do.
bool overlap(const nbo_matrix &a, const nbo_matrix &b)
{
    const uint64_t ea = extent(a), eb = extent(b);
    const uintptr_t pa = (uintptr_t)a.data, pb = (uintptr_t)b.data;
    if (!ea || !eb || pa + ea <= pb || pb + eb <= pa) return false;
    const uint64_t sa = a.stride * size_of(a.dtype), sb = b.stride * size_of(b.dtype);
    if (a.rows > 1 && b.rows > 1 && sa == sb) {
        const uint64_t wa = a.cols * size_of(a.dtype), wb = b.cols * size_of(b.dtype);
        const uint64_t d = pa >= pb ? (pa - pb) % sa : (sa - (pb - pa) % sa) % sa; // a's column in b's rows
        if (d >= wb && d + wa <= sa) return false;
    }
    return true;
}

bool overlap(const nbo_matrix &a, const nbo_ids &ids)
{
    const uintptr_t pa = (uintptr_t)a.data, pb = (uintptr_t)ids.data;
    const uint64_t ea = extent(a), eb = id_bytes(ids);
    return ea && eb && pa + ea > pb && pb + eb > pa;
}

bool same(const nbo_matrix &a, const nbo_matrix &b)
{
    return a.data == b.data && a.dtype == b.dtype && a.rows == b.rows && a.cols == b.cols &&
           (a.rows <= 1 || a.stride == b.stride);
}

void check_address(const nbo_matrix &m, const char *what)
{
    const uint64_t bytes = extent(m);
    if (bytes && pointer_checks_enabled()) check_device_address(m.data, bytes, what, Runtime::get().device());
}

void check_address(const nbo_ids &ids)
{
    if (ids.n && pointer_checks_enabled()) check_device_address(ids.data, id_bytes(ids), "ids", Runtime::get().device());
}

NboUnits units_of(uint64_t rows, uint64_t per_row)
{
    NboUnits u = {};
    u.total = rows * per_row;
    u.per_row = (uint32_t)per_row;
    if (per_row > 1) {
        u.m64 = UINT64_MAX / per_row + 1;
        u.m32 = (uint32_t)(0xFFFFFFFFull / per_row + 1);
        // what the 64-bit reciprocal is exact for
        require(u.total <= UINT64_MAX / per_row, NBO_ERR_TOO_LARGE, "matrix too large for one launch");
    }
    return u;
}

uint32_t grid_of(uint64_t items, uint64_t per_wg)
{
    const uint64_t wgs = (items + per_wg - 1) / per_wg;
    require(wgs <= 0xFFFFFFFFull, NBO_ERR_TOO_LARGE, "matrix too large for one launch");
    return (uint32_t)wgs;
}

// Dropout streams past the caches when its tensors are more than the 256 MB of the last level (bf16, x and
// out: 512 MB 88.5 us without, 85.8 with the hint; f32 with residual, 75 MB: 12.5 without, 14.0 with).
constexpr uint64_t STREAM_BYTES = 256ull << 20;

uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// elements of a unit: 16 bytes of the narrower of the two types
uint64_t unit_elems(int a, int b) { return 16 / std::min(size_of(a), size_of(b)); }

// ---- the gradient's plan -------------------------------------------------------------------

// Ids per piece: as many of 64, 32, 16 as leave SUM_WAVES waves to the chip, or 8: a piece's waves walk it one
// id after the other, and every piece leaves sums to the join (65536 rows of 512 bf16: 52.7 us with 2048 waves, 51.5
// with 4096, 56.7 with 8192; 16384 of 2048: 46.6, 44.4, 47.2).
constexpr uint64_t SUM_WAVES = 4096;
constexpr uint64_t PIECE_MAX = 64, PIECE_MIN = 8;
// Most workgroups of the join, 16 for each compute unit; with more boundaries than that a workgroup looks at
// several (1023 boundaries and 8 slabs each: 13.4 us, one to a workgroup 15.8).
constexpr uint64_t JOIN_WGS = 4096;

// Above either the direct form's matrix is cleared ahead of it, by a launch that does nothing else and fills faster
// (77 MB 14.6 us in one launch, 16.0 in two; 154 MB 28.5 and 26.7; 1051 MB 182 and 161; 131072 rows of 96 bytes 14.2
// and 9.3, 50257 of 512 bytes 9.1 and 9.4).
constexpr uint64_t CLEAR_FIRST_BYTES = 128ull << 20, CLEAR_FIRST_ROWS = 1ull << 16;

// lanes that work on one piece
uint64_t piece_lanes(uint64_t units)
{
    uint64_t l = 1;
    while (l < units && l < 64) l *= 2;
    return l;
}

uint64_t piece_size(uint64_t n, uint64_t units)
{
    const uint64_t lanes = piece_lanes(units), lanes_per_piece = lanes < 64 ? lanes : ceil_div(units, 64) * 64;
    uint64_t p = PIECE_MAX;
    while (p > PIECE_MIN && n / p * lanes_per_piece < SUM_WAVES * 64) p /= 2;
    return p;
}

// Bytes of partial sums that no call over at most max_ids ids and max_cols columns exceeds.  A call has
// two slots of units * unit values, at most cols + 7, for each of its pieces.  There are at most
// ceil(n / 64) of them, or, where the rule above went below 64 ids, fewer than
// 2 * SUM_WAVES * 64 / lanes + 2 (twice as many ids were too few), and a lane's unit has at most 8 values.
uint64_t partial_bound(uint64_t max_ids, uint64_t max_cols)
{
    const uint64_t width = max_cols + 7;
    const uint64_t by_min = ceil_div(max_ids, PIECE_MIN) * width;
    const uint64_t by_rule = std::max(ceil_div(max_ids, PIECE_MAX) * width, 2 * SUM_WAVES * 64 * 8 + 2 * width);
    return 2 * std::min(by_min, by_rule) * 8;
}

int bits_of(uint64_t x)
{
    int b = 0;
    while (x >> b) b++;
    return b;
}

// Into how many ranges, as a power of two, the rows are dealt out: one for each of the 256 compute units, or
// as many as leave at most `keys` to each.
uint32_t range_shift(uint64_t rows, uint64_t keys)
{
    uint32_t shift = 8;
    while (((rows - 1) >> shift) + 1 > keys) shift++;
    return shift;
}

void launch_clear(NboClearArgs c, uint64_t rows)
{
    if (c.grad_stride == c.row_bytes && rows * c.row_bytes >= 16) { // (with no rows to leave alone, whatever their width)
        c.flat_bytes = rows * c.row_bytes;
        c.u.total = ceil_div(c.flat_bytes, 16);
    }
    Runtime::get().launch_folded(K_EMBED_CLEAR, grid_of(c.u.total, NBO_OPS_BLOCK), NBO_OPS_BLOCK, c);
}

// The tokens ordered by rows into (keys, pos) of the workspace; returns which of the two buffers.  With a matrix
// to clear, g.named says afterwards which rows have ids, or is null and it has been cleared.
int launch_order(const nbo_ids &ids, uint64_t rows, nbo_embedding_ws *ws, NboEmbedGradArgs &g)
{
    Runtime &rt = Runtime::get();
    NboOrderArgs a = {};
    a.ids = ids.data;
    a.ids64 = ids.type == NBO_ID_I64;
    a.n = (uint32_t)ids.n;
    a.rows = (uint32_t)rows;
    a.hist = ws->hist;
    a.totals = ws->totals;
    auto deal_out = [&](uint32_t shift) {
        a.shift = shift;
        a.digits = (uint32_t)std::min<uint64_t>(rows, 1ull << shift);
        a.range = (uint32_t)((rows - 1) >> shift) + 1;
        a.named = g.clear.grad ? ws->named : nullptr;
        g.named = a.named;
        g.clear.named_shift = a.shift;
        g.clear.named_range = a.range;
    };
    if (ids.n <= NBO_RANGE_IDS && rows <= NBO_NAMED_ROWS) {
        deal_out(range_shift(rows, NBO_RANGE_KEYS));
        a.keys_out = ws->keys[0];
        a.pos_out = ws->pos[0];
        rt.launch(K_ORDER_RANGE, a.digits, NBO_RANGE_BLOCK, a, NBO_RANGE_BLOCK / 64 * 4 * a.range);
        return 0;
    }
    if (rows <= (uint64_t)NBO_SPLIT_KEYS << NBO_RADIX_BITS) {
        deal_out(range_shift(rows, NBO_SPLIT_KEYS));
        a.tiles = grid_of(ids.n, NBO_SPLIT_TILE);
        a.keys_out = ws->keys[1];
        a.pos_out = ws->pos[1];
        rt.launch(K_ORDER_SPLIT, a.tiles, NBO_RADIX_BLOCK, a);
        a.keys_in = ws->keys[1];
        a.pos_in = ws->pos[1];
        a.keys_out = ws->keys[0];
        a.pos_out = ws->pos[0];
        rt.launch(K_ORDER_MERGE, a.digits, NBO_RANGE_BLOCK, a);
        return 0;
    }
    if (g.clear.grad) launch_clear(g.clear, rows);
    const int bits = bits_of(rows); // (the key of ids outside the table is `rows` itself)
    const int passes = (bits + NBO_RADIX_BITS - 1) / NBO_RADIX_BITS;
    const int per = (bits + passes - 1) / passes;
    a.tiles = grid_of(ids.n, NBO_RADIX_TILE);
    a.digits = 1u << per;
    int to = 0;
    for (int p = 0; p < passes; p++) {
        to = p & 1;
        a.keys_in = p ? ws->keys[1 - to] : nullptr;
        a.pos_in = p ? ws->pos[1 - to] : nullptr;
        a.keys_out = ws->keys[to];
        a.pos_out = ws->pos[to];
        a.shift = (uint32_t)(p * per);
        rt.launch(K_ORDER_HIST, a.tiles, NBO_RADIX_BLOCK, a);
        rt.launch(K_ORDER_SCAN, a.digits, 64, a);
        rt.launch(K_ORDER_SCATTER, a.tiles, NBO_RADIX_BLOCK, a);
    }
    return to;
}

} // namespace

extern "C" {

int nbo_embedding(const nbo_matrix *table, const nbo_ids *ids, const nbo_matrix *add, double scale, const nbo_matrix *out)
{
    return guarded([&] {
        check_form(table, "table");
        check_ids(ids);
        check_form(out, "out");
        check_shape(*out, ids->n, table->cols, "embedding, out");
        int pair = table->dtype; // f32, bf16, f64, f16
        if (table->dtype != out->dtype) {
            require(table->dtype == NBO_DT_F32 && is_half(out->dtype), NBO_ERR_DTYPE,
                    "embedding: out has the table's element type, or bf16 / f16 over an f32 table");
            pair = out->dtype == NBO_DT_BF16 ? 4 : 5;
        }
        if (add) {
            check_form(add, "add");
            check_shape(*add, ids->n, table->cols, "embedding, add");
            require(add->dtype == out->dtype, NBO_ERR_DTYPE, "embedding: add and out differ in element type");
            require(same(*add, *out) || !overlap(*add, *out), NBO_ERR_ARG, "embedding: out overlaps add in part");
        }
        require(!overlap(*table, *out) && !overlap(*out, *ids), NBO_ERR_ARG, "embedding: out overlaps the table or the ids");
        Runtime &rt = Runtime::get();
        if (ids->n == 0 || table->cols == 0) return;
        const OnDevice on(rt.device());
        check_address(*table, "table");
        check_address(*ids);
        if (add && !same(*add, *out)) check_address(*add, "add");
        check_address(*out, "out");
        NboEmbedArgs a = {};
        a.table = table->data;
        a.ids = ids->data;
        a.add = add ? add->data : nullptr;
        a.out = out->data;
        a.table_stride = table->stride * size_of(table->dtype);
        a.add_stride = add ? add->stride * size_of(add->dtype) : 0;
        a.out_stride = out->stride * size_of(out->dtype);
        a.u = units_of(ids->n, ceil_div(table->cols, unit_elems(table->dtype, out->dtype)));
        a.scale = scale;
        a.rows = (uint32_t)table->rows;
        a.cols = (uint32_t)table->cols;
        a.ids64 = ids->type == NBO_ID_I64;
        rt.launch_folded(K_EMBED_BASE + pair, grid_of(a.u.total, NBO_OPS_BLOCK * NBO_EMBED_UNITS), NBO_OPS_BLOCK, a);
    });
}

int nbo_embedding_ws_create(uint64_t max_ids, uint64_t max_cols, nbo_embedding_ws **out)
{
    return guarded([&] {
        require(out != nullptr, NBO_ERR_ARG, "null output pointer");
        *out = nullptr;
        require(max_ids <= MAX_ROWS && max_cols <= MAX_COLS, NBO_ERR_TOO_LARGE, "more than 2^31 - 2 ids or 2^27 columns");
        Runtime &rt = Runtime::get();
        const OnDevice on(rt.device());
        rt.load_operators();
        nbo_embedding_ws *w = new nbo_embedding_ws();
        try {
            w->max_ids = max_ids;
            w->max_cols = max_cols;
            if (max_ids > NBO_EMBED_DIRECT_MAX) { // (the direct form needs none)
                w->partial_bytes = partial_bound(max_ids, max_cols);
                uint64_t total = 0;
                auto piece = [&](uint64_t bytes) {
                    const uint64_t at = total;
                    total += ceil_div(bytes, 256) * 256;
                    return at;
                };
                uint64_t order[4];
                for (uint64_t &o : order) o = piece(max_ids * 4);
                const uint64_t hist = piece(((1ull << NBO_RADIX_BITS) + 1) * ceil_div(max_ids, NBO_SPLIT_TILE) * 4);
                const uint64_t totals = piece(4ull << NBO_RADIX_BITS), named = piece(NBO_NAMED_ROWS);
                const uint64_t partial = piece(w->partial_bytes);
                w->blob = rt.dmalloc(total);
                char *p = (char *)w->blob;
                for (int k = 0; k < 2; k++) {
                    w->keys[k] = (uint32_t *)(p + order[k]);
                    w->pos[k] = (uint32_t *)(p + order[2 + k]);
                }
                w->hist = (uint32_t *)(p + hist);
                w->totals = (uint32_t *)(p + totals);
                w->named = (uint8_t *)(p + named);
                w->partial = p + partial;
            }
            *out = w;
        } catch (...) {
            rt.dfree(w->blob);
            delete w;
            throw;
        }
    });
}

int nbo_embedding_ws_destroy(nbo_embedding_ws *ws)
{
    return guarded([&] {
        if (!ws) return;
        Runtime &rt = Runtime::get();
        const OnDevice on(rt.device());
        rt.sync();
        rt.dfree(ws->blob);
        delete ws;
    });
}

int nbo_embedding_grad(const nbo_matrix *grad_out, const nbo_ids *ids, double scale, int accumulate,
                       const nbo_matrix *grad, nbo_embedding_ws *ws)
{
    return guarded([&] {
        check_form(grad_out, "grad_out");
        check_ids(ids);
        check_form(grad, "grad");
        require(ws != nullptr, NBO_ERR_ARG, "null workspace");
        check_shape(*grad_out, ids->n, grad->cols, "embedding_grad, grad_out");
        int pair = grad->dtype;
        if (grad->dtype != grad_out->dtype) {
            require(grad->dtype == NBO_DT_F32 && is_half(grad_out->dtype), NBO_ERR_DTYPE,
                    "embedding_grad: grad has grad_out's element type, or f32 under bf16 / f16");
            pair = grad_out->dtype == NBO_DT_BF16 ? 4 : 5;
        }
        if (ids->n > ws->max_ids || grad->cols > ws->max_cols)
            fail(NBO_ERR_TOO_LARGE, "embedding_grad: " + std::to_string(ids->n) + " ids of " + std::to_string(grad->cols) +
                                        " columns, the workspace is for " + std::to_string(ws->max_ids) + " of " +
                                        std::to_string(ws->max_cols));
        require(!overlap(*grad, *grad_out) && !overlap(*grad, *ids), NBO_ERR_ARG,
                "embedding_grad: grad overlaps grad_out or the ids");
        Runtime &rt = Runtime::get();
        if (grad->rows == 0 || grad->cols == 0 || (ids->n == 0 && accumulate)) return;
        const OnDevice on(rt.device());
        check_address(*grad_out, "grad_out");
        check_address(*ids);
        check_address(*grad, "grad");
        NboEmbedGradArgs a = {};
        const uint64_t unit = unit_elems(grad->dtype, grad_out->dtype);
        a.dy = grad_out->data;
        a.grad = grad->data;
        a.dy_stride = grad_out->stride * size_of(grad_out->dtype);
        a.grad_stride = grad->stride * size_of(grad->dtype);
        a.scale = scale;
        a.n = (uint32_t)ids->n;
        a.rows = (uint32_t)grad->rows;
        a.cols = (uint32_t)grad->cols;
        a.units = (uint32_t)ceil_div(grad->cols, unit);
        a.slabs = (uint32_t)ceil_div(a.units, 64);
        a.accumulate = accumulate ? 1u : 0u;
        a.ids64 = ids->type == NBO_ID_I64;
        const uint64_t waves_per_wg = NBO_OPS_BLOCK / 64;
        if (!accumulate) {
            a.clear.grad = grad->data;
            a.clear.grad_stride = a.grad_stride;
            a.clear.row_bytes = grad->cols * size_of(grad->dtype);
            a.clear.u = units_of(grad->rows, ceil_div(a.clear.row_bytes, 16));
            if (a.grad_stride == a.clear.row_bytes && a.clear.row_bytes % 16 == 0) a.clear.flat_bytes = grad->rows * a.clear.row_bytes;
        }
        if (ids->n <= NBO_EMBED_DIRECT_MAX) {
            a.ids = ids->data;
            a.sum_wgs = grid_of(ids->n * a.slabs, 1);
            if (a.clear.grad && (grad->rows * a.clear.row_bytes > CLEAR_FIRST_BYTES || grad->rows > CLEAR_FIRST_ROWS)) {
                launch_clear(a.clear, grad->rows);
                a.clear.grad = nullptr;
                if (ids->n == 0) return;
            }
            const uint32_t clear_wgs = a.clear.grad ? grid_of(grad->rows, NBO_CLEAR_ROWS * waves_per_wg) : 0;
            rt.launch_folded(K_EMBED_DIRECT_BASE + pair, grid_of((uint64_t)a.sum_wgs + clear_wgs, 1), NBO_OPS_BLOCK, a);
            return;
        }
        a.piece = (uint32_t)piece_size(ids->n, a.units);
        a.pieces = (uint32_t)ceil_div(ids->n, a.piece);
        a.lanes = (uint32_t)piece_lanes(a.units);
        // (twice, of sums of 4 or 8 bytes)
        const uint64_t need = 2ull * a.pieces * a.units * unit * (grad->dtype == NBO_DT_F64 ? 8 : 4);
        require(need <= ws->partial_bytes, NBO_ERR_TOO_LARGE, "internal: the workspace's partial sums are too small");
        const int order = launch_order(*ids, grad->rows, ws, a);
        a.keys = ws->keys[order];
        a.pos = ws->pos[order];
        a.partial = ws->partial;
        const uint64_t waves = a.lanes == 64 ? (uint64_t)a.pieces * a.slabs : ceil_div(a.pieces, 64 / a.lanes);
        a.sum_wgs = grid_of(waves, waves_per_wg);
        const uint32_t clear_wgs = a.named ? grid_of(a.clear.u.total, NBO_OPS_BLOCK) : 0;
        rt.launch_folded(K_EMBED_SUM_BASE + pair, grid_of((uint64_t)a.sum_wgs + clear_wgs, 1), NBO_OPS_BLOCK, a);
        // (more ids than the direct form takes are at least nine pieces)
        const uint64_t edges = a.pieces - 1;
        a.edges = (uint32_t)std::min<uint64_t>(64, ceil_div(edges * a.slabs, JOIN_WGS));
        rt.launch_folded(K_EMBED_JOIN_BASE + pair, grid_of(ceil_div(edges, a.edges) * a.slabs, 1), NBO_OPS_BLOCK, a);
    });
}

int nbo_rng_create(uint64_t seed, uint64_t step, nbo_rng **out)
{
    return guarded([&] {
        require(out != nullptr, NBO_ERR_ARG, "null output pointer");
        *out = nullptr;
        Runtime &rt = Runtime::get();
        const OnDevice on(rt.device());
        rt.load_operators();
        nbo_rng *r = new nbo_rng();
        try {
            r->dev = (NboRngDev *)rt.dmalloc(sizeof(NboRngDev));
            const NboRngDev s = {seed, step};
            rt.upload(r->dev, &s, sizeof(s));
            *out = r;
        } catch (...) {
            rt.dfree(r->dev);
            delete r;
            throw;
        }
    });
}

int nbo_rng_destroy(nbo_rng *rng)
{
    return guarded([&] {
        if (!rng) return;
        Runtime &rt = Runtime::get();
        const OnDevice on(rt.device());
        rt.sync();
        rt.dfree(rng->dev);
        delete rng;
    });
}

int nbo_rng_state_get(nbo_rng *rng, uint64_t *seed, uint64_t *step)
{
    return guarded([&] {
        require(rng && seed && step, NBO_ERR_ARG, "null generator or output");
        Runtime &rt = Runtime::get();
        const OnDevice on(rt.device());
        NboRngDev s;
        rt.read_back(&s, rng->dev, sizeof(s));
        *seed = s.seed;
        *step = s.step;
    });
}

int nbo_rng_load_state(nbo_rng *rng, uint64_t seed, uint64_t step)
{
    return guarded([&] {
        require(rng != nullptr, NBO_ERR_ARG, "null generator");
        Runtime &rt = Runtime::get();
        const OnDevice on(rt.device());
        const NboRngDev s = {seed, step};
        rt.upload(rng->dev, &s, sizeof(s));
    });
}

int nbo_rng_advance(nbo_rng *rng, uint64_t steps)
{
    return guarded([&] {
        require(rng != nullptr, NBO_ERR_ARG, "null generator");
        Runtime &rt = Runtime::get();
        const OnDevice on(rt.device());
        const NboRngAdvanceArgs a = {rng->dev, steps};
        rt.launch(K_RNG_ADVANCE, 1, 64, a);
    });
}

int nbo_dropout(const nbo_matrix *x, const nbo_matrix *residual, double p, nbo_rng *rng, uint32_t site,
                const nbo_matrix *out)
{
    return guarded([&] {
        check_form(x, "x");
        check_form(out, "out");
        require(rng != nullptr, NBO_ERR_ARG, "null generator");
        require(p >= 0.0 && p <= 1.0, NBO_ERR_ARG, "dropout: p is not in [0, 1]");
        check_shape(*out, x->rows, x->cols, "dropout, out");
        require(x->dtype == out->dtype, NBO_ERR_DTYPE, "dropout: x and out differ in element type");
        require(same(*x, *out) || !overlap(*x, *out), NBO_ERR_ARG, "dropout: out overlaps x in part");
        if (residual) {
            check_form(residual, "residual");
            check_shape(*residual, x->rows, x->cols, "dropout, residual");
            require(residual->dtype == out->dtype, NBO_ERR_DTYPE, "dropout: residual and out differ in element type");
            require(same(*residual, *out) || !overlap(*residual, *out), NBO_ERR_ARG, "dropout: out overlaps residual in part");
        }
        const uint64_t n = x->rows * x->cols;
        require(n <= 1ull << 35, NBO_ERR_TOO_LARGE, "dropout: more than 2^35 elements");
        Runtime &rt = Runtime::get();
        if (n == 0) return;
        const OnDevice on(rt.device());
        check_address(*x, "x");
        if (residual) check_address(*residual, "residual");
        if (!same(*x, *out) && !(residual && same(*residual, *out))) check_address(*out, "out");
        NboDropoutArgs a = {};
        const uint64_t eb = size_of(x->dtype), unit = unit_elems(x->dtype, x->dtype);
        auto adjacent = [](const nbo_matrix &m) { return m.rows <= 1 || m.stride == m.cols; };
        a.x = x->data;
        a.residual = residual ? residual->data : nullptr;
        a.out = out->data;
        a.x_stride = x->stride * eb;
        a.residual_stride = residual ? residual->stride * eb : 0;
        a.out_stride = out->stride * eb;
        a.flat = adjacent(*x) && adjacent(*out) && (!residual || adjacent(*residual)) ? 1u : 0u;
        if (a.flat) a.u.total = ceil_div(n, unit);
        else a.u = units_of(x->rows, ceil_div(x->cols, unit));
        a.rng = rng->dev;
        const uint32_t thr = (uint32_t)std::floor(p * 65536.0 + 0.5);
        a.thr = thr;
        a.scale = thr < 65536 ? 65536.0 / (65536.0 - thr) : 0.0;
        a.n = n;
        a.cols = (uint32_t)x->cols;
        a.site = site;
        a.once = n * eb * (residual ? 3 : 2) > STREAM_BYTES;
        rt.launch_folded(K_DROPOUT_BASE + x->dtype, grid_of(a.u.total, NBO_OPS_BLOCK), NBO_OPS_BLOCK, a);
    });
}

} // extern "C"
