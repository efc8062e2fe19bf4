// Plain-old-data argument blocks shared by the operator kernels (kernels/nbo_ops_kernels.hip) and
// their host side (host/nbo_ops.cpp).  Element type codes are nbo_device_types.h's.
#ifndef NBO_OPS_TYPES_H
#define NBO_OPS_TYPES_H

#include <stdint.h>

// Units per thread of the lookup.
#define NBO_EMBED_UNITS 4
#define NBO_OPS_BLOCK 256u // threads of every operator kernel but the ordering ones

// The generator's state in device memory.
struct NboRngDev {
    uint64_t seed, step;
};

// Rows of `cols` elements cut into units of VEC elements (16 bytes of the 16-bit or wider type, see
// Pair in the kernels), numbered through the matrix: row = unit / per_row.  m32 and m64 are
// ceil(2^32 / per_row) and ceil(2^64 / per_row) (0 for per_row = 1).
struct NboUnits {
    uint64_t total;
    uint64_t m64;
    uint32_t per_row;
    uint32_t m32;
};

struct NboEmbedArgs {
    const void *table;
    const void *ids;
    const void *add; // may be null
    void *out;
    uint64_t table_stride, add_stride, out_stride; // bytes
    NboUnits u;
    double scale;
    uint32_t rows, cols;
    uint32_t ids64;
    uint32_t pad;
};

struct NboDropoutArgs {
    const void *x;
    const void *residual; // may be null
    void *out;
    uint64_t x_stride, residual_stride, out_stride; // bytes
    NboUnits u;
    const NboRngDev *rng;
    double scale;
    uint64_t n;   // elements
    uint32_t cols; // of a row of units; flat matrices are one row
    uint32_t site;
    uint32_t thr; // 0 .. 65536
    uint32_t flat; // rows are adjacent: units run through the matrix
    uint32_t once; // more than the last level of cache holds: stream past it
    uint32_t pad;
};

struct NboRngAdvanceArgs {
    NboRngDev *rng;
    uint64_t steps;
};

// ---- the gradient of the embedding ------------------------------------------------------
// Keys: the ids, with every id outside the table replaced by `rows`; padding comes last.

// Order in one launch, every workgroup reads all ids; threads, and the most ids (they stay in registers) and keys
// per workgroup (LDS: 4 bytes for each wave and key).  The whole gradient of 8192 ids, 512 bf16 columns: 20.1 us, by
// split and merge 22.2; of 4096 ids 18.1 and 21.2.
#define NBO_RANGE_BLOCK 1024u
#define NBO_RANGE_IDS 8192u
#define NBO_RANGE_KEYS 960u
// Radix passes: ids per workgroup and the widest digit.
#define NBO_RADIX_TILE 4096u
#define NBO_RADIX_BLOCK 512u
#define NBO_RADIX_BITS 10u
// Split and merge: ids per tile, and the most keys of a range (LDS of the merge: 4 bytes for each wave and key).
#define NBO_SPLIT_TILE 1024u
#define NBO_SPLIT_KEYS 512u
// Up to this many ids the gradient is one launch that needs no order: as many as every workgroup holds in eight
// registers a lane.  That is the limit, and not where the two ways take the same time: 512 f32 rows of 3 KiB
// 6.6 us, 513 by way of an order 14.1.
#define NBO_EMBED_DIRECT_MAX 512u

// Rows are dealt out to ranges: row v is number v >> shift of range v % 2^shift.
// The matrix to clear, in units of 16 bytes.
#define NBO_CLEAR_ROWS 4u // per wave, in the direct form
struct NboClearArgs {
    void *grad; // null: none
    uint64_t grad_stride, row_bytes;
    uint64_t flat_bytes; // of a matrix whose units follow one another, or 0
    NboUnits u;
    uint32_t named_shift, named_range; // how `named` is laid out: [ranges][named_range] bytes, whether a row has ids
};

// Largest table for which the ordering launches note the rows that have ids (one byte each).  Larger ones are
// cleared as a whole, ahead of the sums.
#define NBO_NAMED_ROWS (NBO_RANGE_KEYS << 11)

struct NboOrderArgs {
    uint8_t *named;        // [ranges][range] or null: whether a row has ids
    const void *ids;       // the caller's (first pass), or null: keys_in / pos_in
    const uint32_t *keys_in, *pos_in;
    uint32_t *keys_out, *pos_out;
    uint32_t *hist;        // [digits][tiles]; of the split: [digits + 1][tiles]
    uint32_t *totals;      // [digits]
    uint32_t n;
    uint32_t rows;
    uint32_t ids64;
    uint32_t tiles;
    uint32_t shift, digits; // radix passes: this pass's digit is (key >> shift) & (digits - 1); otherwise 2^shift
                            // ranges, of which `digits` have rows
    uint32_t range;         // keys per range
    uint32_t pad;
};

struct NboEmbedGradArgs {
    const void *dy;
    void *grad;
    const void *ids;              // the direct form only
    const uint32_t *keys, *pos;   // ordered by rows
    void *partial;                // [pieces][2][units * VEC] sums of rows that span pieces
    uint64_t dy_stride, grad_stride; // bytes
    NboClearArgs clear;
    const uint8_t *named;         // whether a row has ids (null: nothing to clear)
    double scale;
    uint32_t n, rows, cols;
    uint32_t units;               // per row
    uint32_t lanes;               // lanes that work on one piece: 64, or a power of two that holds `units`
    uint32_t slabs;               // waves per piece: 64 units each
    uint32_t piece, pieces;       // ids per piece, pieces
    uint32_t edges;               // boundaries between pieces per workgroup of the join, at most 64
    uint32_t sum_wgs;             // workgroups that add; those behind them clear
    uint32_t accumulate;
    uint32_t ids64;
};

#endif
