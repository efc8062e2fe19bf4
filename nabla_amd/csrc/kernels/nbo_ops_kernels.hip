// gfx950 (CDNA4) kernels of the operators of include/nabla_ops.h: embedding lookup, its gradient,
// and dropout from a counter-based generator.  A code object of its own beside the optimizer's.
//
//   nbo_embed_*        out[t] = add[t] + scale * table[ids[t]]
//   nbo_order_range    the tokens ordered by rows, in one launch (up to 8192 ids)
//   nbo_order_split / _merge             ... in two (more ids)
//   nbo_order_hist / _scan / _scatter    ... by radix passes (tables of more than half a million rows)
//   nbo_embed_clear    zeros everywhere, ahead of the sums: large tables of which few rows are named
//   nbo_embed_sum_*    grad[v] (+)= scale * sum of the rows of dy that name v, in pieces of the order; zeros in the
//                      rows no id names
//   nbo_embed_join_*   ... of the rows whose tokens span pieces
//   nbo_embed_direct_* the whole gradient in one launch, for a few ids
//   nbo_dropout_*      out = residual + kept(x) * scale
//   nbo_rng_advance    step += steps
//
// All of them move bytes and compute little (dropout: some 100 integer operations per 16 bytes), so
// they are organised around 128-bit accesses.  Rows of any width and alignment are cut into units of
// 16 bytes; a row's last unit is moved back so that it ends with the row and is loaded whole, and only
// the elements that no other unit has are stored.  Accesses are at element alignment: global memory
// takes them in one instruction.  Sums and products are f32 (f64 for f64 tensors), rounded to nearest
// once, when a result is stored.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../nbo_device_types.h"
#include "../nbo_ops_types.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));

#define DEV static __device__ __forceinline__
// Addresses arrive as integers; telling the compiler that they are global memory turns flat_*
// accesses into global_* ones.
#define GLOBAL_PTR(type, p) ((__attribute__((address_space(1))) type *)(uintptr_t)(p))

// ---------------------------------------------------------------------------------
// Element types.  A: what sums and products are held in.
template <int E> struct El;
template <> struct El<NBO_F32> {
    typedef float A;
    typedef float Bits;
    typedef f32x4 Vec; // 16 bytes
    DEV A wide(Bits b) { return b; }
    DEV Bits narrow(A x) { return x; }
};
template <> struct El<NBO_F64> {
    typedef double A;
    typedef double Bits;
    typedef f64x2 Vec;
    DEV A wide(Bits b) { return b; }
    DEV Bits narrow(A x) { return x; }
};
template <> struct El<NBO_BF16> {
    typedef float A;
    typedef uint16_t Bits;
    typedef u16x8 Vec;
    DEV A wide(Bits b) { return __uint_as_float((uint32_t)b << 16); }
    DEV Bits narrow(A x) { return __builtin_bit_cast(Bits, (__bf16)x); }
};
template <> struct El<NBO_F16> {
    typedef float A;
    typedef uint16_t Bits;
    typedef u16x8 Vec;
    DEV A wide(Bits b) { return (float)__builtin_bit_cast(_Float16, b); }
    DEV Bits narrow(A x) { return __builtin_bit_cast(Bits, (_Float16)x); }
};

// Loads that are to be in flight together stand outside of branches (what a lane must not use is loaded
// from a place that exists): at the end of a branch that loads, the compiler may wait.

// A unit of V elements of type E as it lies in memory: 16 bytes, or 32 where the other tensor of the
// operator has elements of half the size.
template <int E, int V> struct Unit {
    typedef typename El<E>::Bits Bits;
    typedef typename El<E>::A A;
    enum { SZ = sizeof(Bits), PER = 16 / SZ, N = V * SZ / 16 };
    u32x4 w[N];
    // TINY: the matrix is narrower than a unit, n < V.  ONCE: the bytes are not needed again soon
    template <bool TINY, bool ONCE> __device__ __forceinline__ void load(const char *p, uint32_t n)
    {
        if (!TINY) {
#pragma unroll
            for (int k = 0; k < N; k++)
                w[k] = ONCE ? __builtin_nontemporal_load(GLOBAL_PTR(const u32x4_e, p + 16 * k))
                            : *GLOBAL_PTR(const u32x4_e, p + 16 * k);
        } else {
            A x[V];
#pragma unroll
            for (int j = 0; j < V; j++) x[j] = (uint32_t)j < n ? El<E>::wide(*GLOBAL_PTR(const Bits, p + j * SZ)) : (A)0;
            pack(x);
        }
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int k = 0; k < N; k++) w[k] = 0;
    }
    __device__ __forceinline__ void unpack(A (&x)[V]) const
    {
#pragma unroll
        for (int k = 0; k < N; k++) {
            const typename El<E>::Vec v = __builtin_bit_cast(typename El<E>::Vec, w[k]);
#pragma unroll
            for (int j = 0; j < PER; j++) x[k * PER + j] = El<E>::wide(v[j]);
        }
    }
    __device__ __forceinline__ void pack(const A (&x)[V])
    {
#pragma unroll
        for (int k = 0; k < N; k++) {
            typename El<E>::Vec v;
#pragma unroll
            for (int j = 0; j < PER; j++) v[j] = El<E>::narrow(x[k * PER + j]);
            w[k] = __builtin_bit_cast(u32x4, v);
        }
    }
    // elements skip .. n - 1
    template <bool ONCE> __device__ __forceinline__ void store(char *p, uint32_t skip, uint32_t n) const
    {
        if (skip == 0 && n == V) {
#pragma unroll
            for (int k = 0; k < N; k++) {
                if (ONCE) __builtin_nontemporal_store((u32x4_e)w[k], GLOBAL_PTR(u32x4_e, p + 16 * k));
                else *GLOBAL_PTR(u32x4_e, p + 16 * k) = w[k];
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
            const typename El<E>::Vec v = __builtin_bit_cast(typename El<E>::Vec, w[k]);
#pragma unroll
            for (int j = 0; j < PER; j++)
                if ((uint32_t)(k * PER + j) >= skip && (uint32_t)(k * PER + j) < n)
                    *GLOBAL_PTR(Bits, p + (k * PER + j) * SZ) = v[j];
        }
    }
};

// elements of a unit: 16 bytes of the smaller type
template <int E1, int E2> struct Pair {
    enum {
        S1 = sizeof(typename El<E1>::Bits),
        S2 = sizeof(typename El<E2>::Bits),
        V = 16 / (S1 < S2 ? S1 : S2)
    };
};

// Where unit v of a row of `cols` elements lies: from element c0 on, n elements, of which the first
// `skip` belong to the unit before as well.
struct Span {
    uint32_t c0, skip, n;
};
template <int V> DEV Span unit_span(uint32_t v, uint32_t cols)
{
    Span s;
    if (cols < V) {
        s.c0 = s.skip = 0;
        s.n = cols;
    } else {
        const uint32_t c = v * V;
        s.c0 = c + V <= cols ? c : cols - V;
        s.skip = c - s.c0;
        s.n = V;
    }
    return s;
}

// a launch whose grid the host may have folded into two dimensions
DEV uint32_t folded_workgroup() { return blockIdx.y * gridDim.x + blockIdx.x; }

// (row, unit in the row) of unit `base` + x, x < 1024: base's by the host's 64-bit reciprocal (exact while
// base * per_row < 2^64), x's share by the 32-bit one (exact for these x while per_row < 1024; in longer rows
// x reaches the next row at most)
struct UnitBase {
    uint64_t row;
    uint32_t first; // base's unit within `row`
};
DEV UnitBase unit_base(const NboUnits &u, uint64_t base)
{
    UnitBase b;
    b.row = u.per_row == 1 ? base : __umul64hi(base, u.m64);
    b.first = (uint32_t)(base - b.row * u.per_row);
    return b;
}
DEV void unit_from(const NboUnits &u, const UnitBase &b, uint32_t x, uint32_t *rows_on, uint32_t *v)
{
    const uint32_t y = b.first + x;
    if (u.per_row == 1) *rows_on = y;
    else if (u.per_row < 1024) *rows_on = __umulhi(y, u.m32);
    else *rows_on = y >= u.per_row ? 1u : 0u;
    *v = y - *rows_on * u.per_row;
}
DEV void unit_at(const NboUnits &u, const UnitBase &b, uint32_t x, uint64_t *row, uint32_t *v)
{
    uint32_t on;
    unit_from(u, b, x, &on, v);
    *row = b.row + on;
}

// The ids of U tokens as rows of the table, `rows` for one outside it.  (All loads first, then the keys: a
// branch that used what it loads would wait for it.)
template <int U> DEV void load_keys(const void *ids, uint32_t ids64, const uint64_t (&t)[U], uint32_t rows, uint32_t (&key)[U])
{
    uint64_t id[U];
    if (ids64) {
#pragma unroll
        for (int k = 0; k < U; k++) id[k] = GLOBAL_PTR(const uint64_t, ids)[t[k]];
    } else {
#pragma unroll
        for (int k = 0; k < U; k++) id[k] = GLOBAL_PTR(const uint32_t, ids)[t[k]];
    }
#pragma unroll
    for (int k = 0; k < U; k++) key[k] = id[k] < rows ? (uint32_t)id[k] : rows;
}

// ---------------------------------------------------------------------------------
// The lookup: U units per thread, all ids read, then all rows, then all stores.  Two loads that wait for one
// another, the id and its row, so that what is in flight decides: 65536 rows of 8 KiB with one unit a thread 181 us,
// two 149, four 131 (5.3 TB/s of rows and result; a copy in the best shape 6.65), eight 154.  Rows are kept in the
// caches, for the ids that come again (past them: 176 us), the result is not.
template <int ET, int EO, int U, bool TINY> DEV void embed_body(const NboEmbedArgs &a)
{
    enum { V = Pair<ET, EO>::V, ST = sizeof(typename El<ET>::Bits), SO = sizeof(typename El<EO>::Bits) };
    typedef typename El<EO>::A A;
    const uint64_t base = (uint64_t)folded_workgroup() * (NBO_OPS_BLOCK * U);
    if (base >= a.u.total) return; // the unused end of a folded grid
    const UnitBase b = unit_base(a.u, base);
    uint64_t t[U];
    uint32_t v[U], key[U];
    bool on[U];
#pragma unroll
    for (int k = 0; k < U; k++) {
        const uint32_t x = threadIdx.x + k * NBO_OPS_BLOCK;
        on[k] = base + x < a.u.total;
        // (what is beyond the end looks at the first unit again and stores nothing)
        unit_at(a.u, b, on[k] ? x : 0, &t[k], &v[k]);
    }
    load_keys<U>(a.ids, a.ids64, t, a.rows, key);
    Unit<ET, V> row[U];
    Unit<EO, V> add[U];
    if (a.rows > 0) {
#pragma unroll
        for (int k = 0; k < U; k++) { // (padding looks at row 0)
            const Span s = unit_span<V>(v[k], a.cols);
            const uint64_t r = key[k] < a.rows ? key[k] : 0;
            row[k].template load<TINY, false>((const char *)a.table + r * a.table_stride + (uint64_t)s.c0 * ST, s.n);
        }
    } else {
#pragma unroll
        for (int k = 0; k < U; k++) row[k].clear();
    }
    if (a.add) {
#pragma unroll
        for (int k = 0; k < U; k++) {
            const Span s = unit_span<V>(v[k], a.cols);
            add[k].template load<TINY, false>((const char *)a.add + t[k] * a.add_stride + (uint64_t)s.c0 * SO, s.n);
        }
    }
    const A scale = (A)a.scale;
#pragma unroll
    for (int k = 0; k < U; k++) {
        if (!on[k]) continue;
        const Span s = unit_span<V>(v[k], a.cols);
        A x[V];
        row[k].unpack(x);
        // (padding is zero whatever the scale is)
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = key[k] < a.rows ? x[j] * scale : (A)0;
        if (a.add) {
            A y[V];
            add[k].unpack(y);
#pragma unroll
            for (int j = 0; j < V; j++) x[j] = y[j] + x[j];
        }
        Unit<EO, V> o;
        o.pack(x);
        o.template store<true>((char *)a.out + t[k] * a.out_stride + (uint64_t)s.c0 * SO, s.skip, s.n);
    }
}

#define NBO_EMBED_KERNEL(name, ET, EO)                                                      \
    extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void name(const NboEmbedArgs a)  \
    {                                                                                       \
        if (a.cols >= (uint32_t)Pair<ET, EO>::V) embed_body<ET, EO, NBO_EMBED_UNITS, false>(a); \
        else embed_body<ET, EO, NBO_EMBED_UNITS, true>(a);                                  \
    }
NBO_EMBED_KERNEL(nbo_embed_f32, NBO_F32, NBO_F32)
NBO_EMBED_KERNEL(nbo_embed_bf16, NBO_BF16, NBO_BF16)
NBO_EMBED_KERNEL(nbo_embed_f64, NBO_F64, NBO_F64)
NBO_EMBED_KERNEL(nbo_embed_f16, NBO_F16, NBO_F16)
NBO_EMBED_KERNEL(nbo_embed_f32_bf16, NBO_F32, NBO_BF16)
NBO_EMBED_KERNEL(nbo_embed_f32_f16, NBO_F32, NBO_F16)

// inclusive sum over the wave
DEV uint32_t wave_scan(uint32_t x)
{
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const uint32_t y = __shfl_up(x, s);
        if (lane >= (uint32_t)s) x += y;
    }
    return x;
}

// ---------------------------------------------------------------------------------
// The order.  All that the sums need is that the tokens of one row are adjacent and in their own order, so
// rows are dealt out to 2^shift ranges, row v to range v % 2^shift: ids that are close to one another (a
// vocabulary sorted by frequency, positions) are spread over all ranges.  Ranges come in order, within a range the
// rows, within a row its tokens; padding takes no part, and the places behind the last token hold its key.
// (With ranges of adjacent rows the merge of 65536 ids, log-uniform over 131072 rows in order of frequency, took
// 57 us instead of 13.)  Where most ids are one row, one workgroup does most of the work, at the 25 GB/s that one
// compute unit reads: 65536 ids of one row 45 us.
//
// In one launch: every workgroup owns a range, reads all ids and puts those of its range to their places.
// Nothing passes between workgroups: how many ids come before the range is counted on the way.  Within the
// range an id's place is its key's start, the ids of that key which earlier waves hold (each wave has a run of
// the ids), and those its own wave has seen.  The ids stay in registers from the first look at them to the
// last.  8192 ids: 7.3 us, bound by latency and by the instructions that every workgroup spends on every id.

// For a block of 64 ids of which the lanes in `left` (not empty) count: adds to mine[r] how many lanes hold
// each r.  The lanes that hold what the first one holds are counted as one: an addition to one LDS word takes
// a turn for every lane, and a hot row fills whole blocks.
DEV void count_keys(uint32_t *mine, uint32_t r, uint64_t left)
{
    const uint32_t lane = threadIdx.x & 63u;
    const int first = __builtin_ctzll(left);
    const uint64_t m = left & __builtin_amdgcn_ballot_w64(r == (uint32_t)__builtin_amdgcn_readlane(r, first));
    if ((int)lane == first) atomicAdd(&mine[r], (uint32_t)__popcll(m));
    if ((left & ~m) >> lane & 1) atomicAdd(&mine[r], 1u);
}

DEV uint32_t lanes_before(uint64_t m)
{
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// ... and with mine[r] the place of the next id that has r (r < 2^bits): each lane's place, in the order of
// the lanes.  The counters are one wave's own, so nothing else moves them.  First the lanes that hold what
// the first one holds (all of them, where a row is hot); one or two more one by one; more than that
// together: who holds the same r is found bit by bit.
DEV uint32_t place_keys(uint32_t *mine, uint32_t r, uint64_t left, uint32_t bits)
{
    const uint32_t lane = threadIdx.x & 63u;
    const int first = __builtin_ctzll(left);
    uint64_t same = left & __builtin_amdgcn_ballot_w64(r == (uint32_t)__builtin_amdgcn_readlane(r, first));
    uint32_t at = 0;
    if ((int)lane == first) at = atomicAdd(&mine[r], (uint32_t)__popcll(same));
    const uint32_t next = __builtin_amdgcn_readlane(at, first);
    if (same >> lane & 1) at = next + lanes_before(same);
    left &= ~same;
    if (__popcll(left) <= 2) {
        for (; left; left &= left - 1)
            if ((int)lane == __builtin_ctzll(left)) at = atomicAdd(&mine[r], 1u);
        return at;
    }
    const bool on = left >> lane & 1;
    same = left;
    for (uint32_t b = 0; b < bits; b++) {
        const uint64_t m = __builtin_amdgcn_ballot_w64((r >> b & 1) != 0);
        same &= (r >> b & 1) ? m : ~m;
    }
    const uint32_t ahead = lanes_before(same);
    uint32_t start = 0;
    if (on && ahead == 0) start = atomicAdd(&mine[r], (uint32_t)__popcll(same));
    start = __shfl(start, on ? __builtin_ctzll(same) : 0);
    return on ? start + ahead : at;
}

// a workgroup's sum: one term per wave, to be added up behind a barrier
template <int WAVES> DEV void leave_sum(uint32_t x, uint32_t (&terms)[WAVES])
{
#pragma unroll
    for (int s = 32; s >= 1; s /= 2) x += __shfl_xor(x, s);
    if ((threadIdx.x & 63u) == 0) terms[threadIdx.x >> 6] = x;
}
template <int WAVES> DEV uint32_t total_of(const uint32_t (&terms)[WAVES])
{
    uint32_t x = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) x += terms[w];
    return x;
}

// count[WAVES][range], each wave's number of ids of each key, becomes where the wave's first one goes:
// behind the ids of the ranges before (wbelow: one term per wave), the smaller keys, the waves before.
// One thread per key; range is at most the workgroup's size.  Notes in a.named which rows of the table have
// ids, range by range.
template <int WAVES> DEV void starts_of_keys(const NboOrderArgs &a, uint32_t *count, uint32_t (&wsum)[WAVES],
                                             const uint32_t (&wbelow)[WAVES])
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, range = a.range;
    __syncthreads();
    uint32_t c[WAVES], total = 0;
    if (threadIdx.x < range)
#pragma unroll
        for (int w = 0; w < WAVES; w++) total += c[w] = count[w * range + threadIdx.x];
    if (a.named && threadIdx.x < range) GLOBAL_PTR(uint8_t, a.named)[(uint64_t)blockIdx.x * range + threadIdx.x] = total > 0;
    const uint32_t up = wave_scan(total);
    if (lane == 63) wsum[wave] = up;
    __syncthreads();
    uint32_t at = up - total + total_of<WAVES>(wbelow);
#pragma unroll
    for (int w = 0; w < WAVES; w++)
        if ((uint32_t)w < wave) at += wsum[w];
    if (threadIdx.x < range)
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            count[w * range + threadIdx.x] = at;
            at += c[w];
        }
    __syncthreads();
}

// the padding's key behind the last of the `valid` ids, workgroup wg's share of wgs
DEV void fill_padding(const NboOrderArgs &a, uint32_t valid, uint32_t wg, uint32_t wgs)
{
    for (uint64_t i = (uint64_t)valid + wg * NBO_RANGE_BLOCK + threadIdx.x; i < a.n; i += wgs * NBO_RANGE_BLOCK) {
        GLOBAL_PTR(uint32_t, a.keys_out)[i] = a.rows;
        GLOBAL_PTR(uint32_t, a.pos_out)[i] = 0;
    }
}

// Zeros in `bytes` bytes (an even number) at an even address, by a whole wave: two bytes at a time up to
// the first 16-byte boundary and behind the last.
DEV void clear_bytes(char *p, uint64_t bytes)
{
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t to_boundary = (16u - (uint32_t)((uintptr_t)p & 15u)) & 15u;
    const uint64_t head = to_boundary < bytes ? to_boundary : bytes, nvec = (bytes - head) / 16, tail = head + nvec * 16;
    const u32x4 z = 0;
    char *v = p + head;
#pragma unroll 4
    for (uint64_t i = lane; i < nvec; i += 64) __builtin_nontemporal_store(z, GLOBAL_PTR(u32x4, v + i * 16));
    if (lane * 2 < head) *GLOBAL_PTR(uint16_t, p + lane * 2) = 0;
    if (lane * 2 < bytes - tail) *GLOBAL_PTR(uint16_t, p + tail + lane * 2) = 0;
}

// Zeros in the rows first .. first + count - 1 (count <= 64) whose bit in `named` is not set.  Rows that are
// adjacent in memory are cleared as one run.
DEV void clear_rows(const NboClearArgs &c, uint64_t first, uint32_t count, uint64_t named)
{
    uint64_t left = ~named & (count < 64 ? (1ull << count) - 1 : ~0ull);
    while (left) {
        const uint32_t r = __builtin_ctzll(left);
        const uint64_t run = ~(left >> r); // bit k: row r + k is not to be cleared
        uint32_t k = c.grad_stride == c.row_bytes ? (run ? (uint32_t)__builtin_ctzll(run) : 64u) : 1u;
        clear_bytes((char *)c.grad + (first + r) * c.grad_stride, k * c.row_bytes);
        left = r + k < 64 ? left >> (r + k) << (r + k) : 0;
    }
}

extern "C" __global__ __launch_bounds__(NBO_RANGE_BLOCK) void nbo_order_range(const NboOrderArgs a)
{
    enum { WAVES = NBO_RANGE_BLOCK / 64, U = NBO_RANGE_IDS / NBO_RANGE_BLOCK };
    extern __shared__ uint32_t count[]; // [WAVES][range]
    __shared__ uint32_t wsum[WAVES], wbelow[WAVES];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t blocks = (a.n + 63) / 64, per = (blocks + WAVES - 1) / WAVES; // blocks of 64 ids per wave, at most U
    const uint32_t first = wave * per * 64 + lane, mask = (1u << a.shift) - 1;
    const uint32_t end = (wave + 1) * per * 64 < a.n ? (wave + 1) * per * 64 : a.n; // of the wave's run
    uint64_t t[U];
    uint32_t key[U];
#pragma unroll
    for (int u = 0; u < U; u++) { // (behind the wave's or the last id: that one again)
        const uint32_t i = first + ((uint32_t)u < per ? u : per - 1) * 64;
        t[u] = i < a.n ? i : a.n - 1;
    }
    load_keys<U>(a.ids, a.ids64, t, a.rows, key);
    for (uint32_t i = threadIdx.x; i < WAVES * a.range; i += NBO_RANGE_BLOCK) count[i] = 0;
    __syncthreads();
    uint32_t *mine = count + wave * a.range;
    uint32_t below = 0; // the wave's ids of the ranges before
    uint64_t in[U];     // the lanes whose ids are in the range
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint64_t takes_part = __builtin_amdgcn_ballot_w64(first + u * 64 < end) & __builtin_amdgcn_ballot_w64(key[u] < a.rows);
        below += (uint32_t)__popcll(takes_part & __builtin_amdgcn_ballot_w64((key[u] & mask) < blockIdx.x));
        in[u] = takes_part & __builtin_amdgcn_ballot_w64((key[u] & mask) == blockIdx.x);
        key[u] >>= a.shift;
        if (in[u]) count_keys(mine, key[u], in[u]);
    }
    if (lane == 0) wbelow[wave] = below;
    starts_of_keys<WAVES>(a, count, wsum, wbelow);
    const uint32_t bits = 32 - __builtin_clz((a.range - 1) | 1);
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (!in[u]) continue;
        const uint32_t at = place_keys(mine, key[u], in[u], bits);
        if (in[u] >> lane & 1) {
            GLOBAL_PTR(uint32_t, a.keys_out)[at] = key[u] << a.shift | blockIdx.x;
            GLOBAL_PTR(uint32_t, a.pos_out)[at] = first + u * 64;
        }
    }
    if (blockIdx.x == gridDim.x - 1) fill_padding(a, total_of<WAVES>(wbelow) + total_of<WAVES>(wsum), 0, 1);
}

// ---------------------------------------------------------------------------------
// Table order by stable radix passes of up to ten bits, least significant first, for tables with more rows than
// the ranges hold.  Per pass: how often each digit occurs in each tile; the running sums over the tiles, per
// digit; every id to its place.  65536 ids: 43 us in two passes, each three launches that wait for each other.
template <int N> DEV void order_keys(const NboOrderArgs &a, const uint64_t (&t)[N], uint32_t (&key)[N])
{
    if (!a.keys_in) {
        load_keys<N>(a.ids, a.ids64, t, a.rows, key);
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) key[k] = GLOBAL_PTR(const uint32_t, a.keys_in)[t[k]];
    }
}

extern "C" __global__ __launch_bounds__(NBO_RADIX_BLOCK) void nbo_order_hist(const NboOrderArgs a)
{
    enum { ROWS = NBO_RADIX_TILE / NBO_RADIX_BLOCK };
    __shared__ uint32_t count[1u << NBO_RADIX_BITS];
    for (uint32_t d = threadIdx.x; d < a.digits; d += NBO_RADIX_BLOCK) count[d] = 0;
    const uint32_t first = blockIdx.x * NBO_RADIX_TILE + threadIdx.x;
    uint64_t t[ROWS];
    uint32_t key[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) t[r] = first + r * NBO_RADIX_BLOCK < a.n ? first + r * NBO_RADIX_BLOCK : a.n - 1;
    order_keys<ROWS>(a, t, key);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const uint64_t on = __builtin_amdgcn_ballot_w64(first + r * NBO_RADIX_BLOCK < a.n);
        if (on) count_keys(count, (key[r] >> a.shift) & (a.digits - 1), on);
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < a.digits; d += NBO_RADIX_BLOCK)
        GLOBAL_PTR(uint32_t, a.hist)[(uint64_t)d * a.tiles + blockIdx.x] = count[d];
}

// one wave per digit
extern "C" __global__ __launch_bounds__(64) void nbo_order_scan(const NboOrderArgs a)
{
    auto *h = GLOBAL_PTR(uint32_t, a.hist) + (uint64_t)blockIdx.x * a.tiles;
    uint32_t sum = 0;
    for (uint32_t i = 0; i < a.tiles; i += 64) {
        const uint32_t j = i + threadIdx.x;
        const uint32_t x = j < a.tiles ? h[j] : 0;
        const uint32_t up = wave_scan(x);
        if (j < a.tiles) h[j] = sum + up - x;
        sum += __shfl(up, 63);
    }
    if (threadIdx.x == 0) GLOBAL_PTR(uint32_t, a.totals)[blockIdx.x] = sum;
}

// For the ROWS rows of 64 ids that a wave takes in order, with digits d: how many ids of its digit come
// before each in the wave, and in mine[digit] how many there are.
template <int ROWS> DEV void rank_digits(uint32_t *mine, const uint32_t (&d)[ROWS], const bool (&on)[ROWS], uint32_t digits,
                                         uint32_t (&rank)[ROWS])
{
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        uint64_t same = __builtin_amdgcn_ballot_w64(on[r]);
        for (uint32_t bit = 1; bit < digits; bit <<= 1) { // lanes with the same digit
            const uint64_t m = __builtin_amdgcn_ballot_w64((d[r] & bit) != 0);
            same &= (d[r] & bit) ? m : ~m;
        }
        const uint32_t ahead = lanes_before(same);
        uint32_t seen = 0;
        if (on[r] && ahead == 0) seen = atomicAdd(&mine[d[r]], (uint32_t)__popcll(same)); // (the wave's own counter)
        rank[r] = __shfl(seen, on[r] ? __builtin_ctzll(same) : 0) + ahead;
    }
}

// exclusive sums over a workgroup of NBO_RADIX_BLOCK threads
DEV uint32_t block_starts(uint32_t x, uint32_t (&wsum)[NBO_RADIX_BLOCK / 64])
{
    const uint32_t wave = threadIdx.x >> 6, up = wave_scan(x);
    if ((threadIdx.x & 63u) == 63) wsum[wave] = up;
    __syncthreads();
    uint32_t below = up - x;
    for (uint32_t w = 0; w < wave; w++) below += wsum[w];
    return below;
}

extern "C" __global__ __launch_bounds__(NBO_RADIX_BLOCK) void nbo_order_scatter(const NboOrderArgs a)
{
    enum { WAVES = NBO_RADIX_BLOCK / 64, ROWS = NBO_RADIX_TILE / NBO_RADIX_BLOCK };
    __shared__ uint32_t count[WAVES][1u << NBO_RADIX_BITS]; // per wave, then: where the wave's next one goes
    __shared__ uint32_t wsum[WAVES];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t d = threadIdx.x; d < a.digits; d += NBO_RADIX_BLOCK)
#pragma unroll
        for (int w = 0; w < WAVES; w++) count[w][d] = 0;
    const uint32_t first = blockIdx.x * NBO_RADIX_TILE + wave * (ROWS * 64) + lane;
    uint32_t key[ROWS], pos[ROWS], rank[ROWS], digit[ROWS];
    uint64_t t[ROWS];
    bool on[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        on[r] = first + r * 64 < a.n;
        t[r] = on[r] ? first + r * 64 : a.n - 1;
        pos[r] = first + r * 64;
    }
    order_keys<ROWS>(a, t, key);
    if (a.pos_in) {
#pragma unroll
        for (int r = 0; r < ROWS; r++) pos[r] = GLOBAL_PTR(const uint32_t, a.pos_in)[t[r]];
    }
#pragma unroll
    for (int r = 0; r < ROWS; r++) digit[r] = (key[r] >> a.shift) & (a.digits - 1);
    __syncthreads();
    rank_digits<ROWS>(count[wave], digit, on, a.digits, rank);
    __syncthreads();
    // where each digit starts: the digits below it, the tiles before this one, the waves before each
    const uint32_t per = (a.digits + NBO_RADIX_BLOCK - 1) / NBO_RADIX_BLOCK; // at most 2
    uint32_t tot[2] = {0, 0};
    for (uint32_t k = 0; k < per; k++) {
        const uint32_t d = threadIdx.x * per + k;
        if (d < a.digits) tot[k] = GLOBAL_PTR(const uint32_t, a.totals)[d];
    }
    uint32_t below = block_starts(tot[0] + tot[1], wsum);
    for (uint32_t k = 0; k < per; k++) {
        const uint32_t d = threadIdx.x * per + k;
        if (d >= a.digits) break;
        uint32_t at = below + GLOBAL_PTR(const uint32_t, a.hist)[(uint64_t)d * a.tiles + blockIdx.x];
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const uint32_t c = count[w][d];
            count[w][d] = at;
            at += c;
        }
        below += tot[k];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; r++)
        if (on[r]) {
            const uint32_t at = count[wave][digit[r]] + rank[r];
            GLOBAL_PTR(uint32_t, a.keys_out)[at] = key[r];
            GLOBAL_PTR(uint32_t, a.pos_out)[at] = pos[r];
        }
}

// ---------------------------------------------------------------------------------
// The same order in two launches: every tile puts its ids in the order of the ranges, in place, and notes
// where each range starts; then one workgroup per range collects it from all tiles and orders it as
// nbo_order_range does.  What lies before the range is the sum of the tiles' starts.  Every id is moved twice
// however many there are: 16384 ids 4.7 + 5.3 us, 65536 4.8 + 9.8, bound by latency (five loads and stores one
// after the other).
extern "C" __global__ __launch_bounds__(NBO_RADIX_BLOCK) void nbo_order_split(const NboOrderArgs a)
{
    enum { WAVES = NBO_RADIX_BLOCK / 64, ROWS = NBO_SPLIT_TILE / NBO_RADIX_BLOCK };
    __shared__ uint32_t count[WAVES][1u << NBO_RADIX_BITS];
    __shared__ uint32_t wsum[WAVES];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t d = threadIdx.x; d < a.digits; d += NBO_RADIX_BLOCK)
#pragma unroll
        for (int w = 0; w < WAVES; w++) count[w][d] = 0;
    const uint32_t tile = blockIdx.x * NBO_SPLIT_TILE, first = tile + wave * (ROWS * 64) + lane;
    uint32_t key[ROWS], rank[ROWS], digit[ROWS];
    uint64_t t[ROWS];
    bool on[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        on[r] = first + r * 64 < a.n;
        t[r] = on[r] ? first + r * 64 : a.n - 1;
    }
    load_keys<ROWS>(a.ids, a.ids64, t, a.rows, key);
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        on[r] = on[r] && key[r] < a.rows; // padding is left out
        digit[r] = on[r] ? key[r] & ((1u << a.shift) - 1) : 0;
    }
    __syncthreads();
    rank_digits<ROWS>(count[wave], digit, on, a.digits, rank);
    __syncthreads();
    uint32_t tot[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t d = threadIdx.x * 2 + k;
        if (d < a.digits)
#pragma unroll
            for (int w = 0; w < WAVES; w++) tot[k] += count[w][d];
    }
    uint32_t at = block_starts(tot[0] + tot[1], wsum);
    if (threadIdx.x == NBO_RADIX_BLOCK - 1) // where a range behind the last one would start: the tile's ids
        GLOBAL_PTR(uint32_t, a.hist)[(uint64_t)a.digits * a.tiles + blockIdx.x] = at + tot[0] + tot[1];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t d = threadIdx.x * 2 + k;
        if (d >= a.digits) break;
        GLOBAL_PTR(uint32_t, a.hist)[(uint64_t)d * a.tiles + blockIdx.x] = at;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const uint32_t c = count[w][d];
            count[w][d] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; r++)
        if (on[r]) {
            const uint32_t i = tile + count[wave][digit[r]] + rank[r];
            GLOBAL_PTR(uint32_t, a.keys_out)[i] = key[r];
            GLOBAL_PTR(uint32_t, a.pos_out)[i] = first + r * 64;
        }
}

extern "C" __global__ __launch_bounds__(NBO_RANGE_BLOCK) void nbo_order_merge(const NboOrderArgs a)
{
    enum { WAVES = NBO_RANGE_BLOCK / 64, U = 4 };
    __shared__ uint32_t count[WAVES * NBO_SPLIT_KEYS];
    __shared__ uint32_t wsum[WAVES], wbelow[WAVES], wvalid[WAVES];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t bits = 32 - __builtin_clz((a.range - 1) | 1);
    auto *h = GLOBAL_PTR(const uint32_t, a.hist) + (uint64_t)blockIdx.x * a.tiles;
    auto *keys = GLOBAL_PTR(const uint32_t, a.keys_in);
    auto *poss = GLOBAL_PTR(const uint32_t, a.pos_in);
    const uint32_t per = (a.tiles + WAVES - 1) / WAVES;
    const uint32_t from = wave * per, to = from + per < a.tiles ? from + per : a.tiles;
    auto *ends = GLOBAL_PTR(const uint32_t, a.hist) + (uint64_t)a.digits * a.tiles; // ids that count, per tile
    // (where the wave's first segments lie is asked for together with the sums' terms)
    auto tile_at = [&](uint32_t t0) { return t0 + (lane & 3u) < a.tiles ? t0 + (lane & 3u) : a.tiles - 1; };
    const uint32_t first_start = h[tile_at(from)], first_end = h[a.tiles + tile_at(from)];
    uint32_t below = 0, valid = 0;
    for (uint32_t t = threadIdx.x; t < a.tiles; t += NBO_RANGE_BLOCK) {
        below += h[t];
        valid += ends[t];
    }
    for (uint32_t i = threadIdx.x; i < WAVES * a.range; i += NBO_RANGE_BLOCK) count[i] = 0;
    uint32_t *mine = count + wave * a.range;
    leave_sum<WAVES>(valid, wvalid);
    leave_sum<WAVES>(below, wbelow);
    // The wave's tiles in order, four at a time: the first 64 ids of the range in each of the four are asked
    // for together, with their places, and kept where there is but one such group (up to 64 tiles)
    uint32_t at[U], len[U], key[U], pos[U];
    auto fetch = [&](uint32_t t0, uint32_t start, uint32_t end) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t s = __builtin_amdgcn_readlane(start, u);
            len[u] = t0 + u < to ? __builtin_amdgcn_readlane(end, u) - s : 0;
            at[u] = (t0 + u) * NBO_SPLIT_TILE + s;
        }
#pragma unroll
        for (int u = 0; u < U; u++) { // (behind the segment: its first id again, or the last of all)
            const uint32_t p = at[u] + (lane < len[u] ? lane : 0), q = p < a.n ? p : a.n - 1;
            key[u] = keys[q] >> a.shift;
            pos[u] = poss[q];
        }
    };
    auto place = [&](uint32_t r, uint32_t p, uint64_t in) {
        const uint32_t to_at = place_keys(mine, r, in, bits);
        if (in >> lane & 1) {
            GLOBAL_PTR(uint32_t, a.keys_out)[to_at] = r << a.shift | blockIdx.x;
            GLOBAL_PTR(uint32_t, a.pos_out)[to_at] = p;
        }
    };
    // what a segment has behind its first 64 (a hot row), again four blocks at a time
    auto behind = [&](uint32_t first, uint32_t n, auto &&each) {
        for (uint32_t o = 64; o < n; o += 64 * U) {
            uint32_t k[U], p[U];
#pragma unroll
            for (int j = 0; j < U; j++) {
                const uint32_t q = first + (o + j * 64 + lane < n ? o + j * 64 + lane : 0);
                k[j] = keys[q] >> a.shift;
                p[j] = poss[q];
            }
#pragma unroll
            for (int j = 0; j < U; j++)
                if (o + j * 64 < n) each(k[j], p[j], __builtin_amdgcn_ballot_w64(o + j * 64 + lane < n));
        }
    };
    if (from < to) fetch(from, first_start, first_end);
    __syncthreads();
    for (uint32_t t0 = from; t0 < to; t0 += U) {
        if (t0 > from) fetch(t0, h[tile_at(t0)], h[a.tiles + tile_at(t0)]);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (len[u] == 0) continue;
            count_keys(mine, key[u], __builtin_amdgcn_ballot_w64(lane < len[u]));
            behind(at[u], len[u], [&](uint32_t r, uint32_t, uint64_t in) { count_keys(mine, r, in); });
        }
    }
    starts_of_keys<WAVES>(a, count, wsum, wbelow);
    for (uint32_t t0 = from; t0 < to; t0 += U) {
        if (per > U) fetch(t0, h[tile_at(t0)], h[a.tiles + tile_at(t0)]);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (len[u] == 0) continue;
            place(key[u], pos[u], __builtin_amdgcn_ballot_w64(lane < len[u]));
            behind(at[u], len[u], place);
        }
    }
    fill_padding(a, total_of<WAVES>(wvalid), blockIdx.x, a.digits);
}

// ---------------------------------------------------------------------------------
// The sums.  The order is cut into pieces of a.piece tokens; `lanes` lanes, one unit of the row each,
// walk a piece and add up the rows of dy.  A row of the table all of whose tokens lie in the piece is
// finished there; the sums of one that began in an earlier piece or goes on into the next are left in
// the piece's two slots, for the join.  So a row that half the batch names is added up by many
// waves, and in the same order of additions on every run.  Bound by memory: 65536 bf16 rows of 8 KiB into 128256,
// with the zeros in the other rows, 276 us, 5.6 TB/s.
template <int EG> DEV char *grad_at(const NboEmbedGradArgs &a, uint32_t key, const Span &s)
{
    return (char *)a.grad + key * a.grad_stride + (uint64_t)s.c0 * sizeof(typename El<EG>::Bits);
}
// A finished sum into its row; `g`, when accumulating, is what was there (asked for ahead of the sum).
template <int EG, int V> DEV void finish_row(const NboEmbedGradArgs &a, uint32_t key, const Span &s, Unit<EG, V> &g,
                                             typename El<EG>::A (&x)[V])
{
    typedef typename El<EG>::A A;
    const A scale = (A)a.scale;
    if (a.accumulate) {
        A y[V];
        g.unpack(y);
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = y[j] + scale * x[j];
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = scale * x[j];
    }
    g.pack(x);
    g.template store<true>(grad_at<EG>(a, key, s), s.skip, s.n);
}
template <int EG, int V, bool TINY> DEV void add_to_grad(const NboEmbedGradArgs &a, uint32_t key, const Span &s,
                                                         typename El<EG>::A (&x)[V])
{
    Unit<EG, V> g;
    if (a.accumulate) g.template load<TINY, false>(grad_at<EG>(a, key, s), s.n);
    finish_row<EG, V>(a, key, s, g, x);
}

enum { SLOT_HEAD = 0, SLOT_TAIL = 1 }; // began in an earlier piece / goes on into the next only
template <typename A, int V> DEV char *slot_at(const NboEmbedGradArgs &a, uint32_t piece, uint32_t slot, uint32_t v)
{
    return (char *)a.partial + (((uint64_t)piece * 2 + slot) * a.units + v) * (V * sizeof(A));
}
template <typename A, int V> DEV void store_slot(char *p, const A (&x)[V])
{
#pragma unroll
    for (int j = 0; j < V; j += 16 / (int)sizeof(A)) {
        u32x4 w;
        __builtin_memcpy(&w, &x[j], 16);
        *GLOBAL_PTR(u32x4, p + j * sizeof(A)) = w;
    }
}
template <typename A, int V> DEV void load_slot(const char *p, A (&x)[V])
{
#pragma unroll
    for (int j = 0; j < V; j += 16 / (int)sizeof(A)) {
        const u32x4 w = *GLOBAL_PTR(const u32x4, p + j * sizeof(A));
        __builtin_memcpy(&x[j], &w, 16);
    }
}

// One piece by `lanes` < 64 lanes, for rows of few units: several pieces to a wave.  65536 rows of 48 bf16 take
// 13 us, the latency of 8 tokens one after the other.  (Eight tokens and their rows of the table asked for
// together take 10, but 157 registers instead of 69, and then the clears that share this kernel are slower
// everywhere: 128256 rows of 8 KiB 375 us instead of 282.)
template <int ED, int EG, bool TINY> DEV void sum_narrow(const NboEmbedGradArgs &a, uint32_t wave)
{
    enum { V = Pair<ED, EG>::V, SD = sizeof(typename El<ED>::Bits), U = 4 };
    typedef typename El<EG>::A A;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t piece = wave * (64 / a.lanes) + lane / a.lanes, v = lane % a.lanes;
    if (piece >= a.pieces || v >= a.units) return;
    const Span s = unit_span<V>(v, a.cols);
    const uint32_t from = piece * a.piece, to = a.n - from < a.piece ? a.n : from + a.piece;
    auto *keys = GLOBAL_PTR(const uint32_t, a.keys);
    auto *pos = GLOBAL_PTR(const uint32_t, a.pos);
    uint32_t cur = keys[from];
    if (cur >= a.rows) return; // nothing but padding
    bool head = from > 0 && keys[from - 1] == cur;
    A acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = (A)0;
    for (uint32_t i = from; i < to; i += U) {
        uint32_t key[U], row[U];
        Unit<ED, V> d[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t j = i + u < to ? i + u : to - 1;
            key[u] = keys[j];
            row[u] = pos[j];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            d[u].template load<TINY, true>((const char *)a.dy + row[u] * a.dy_stride + (uint64_t)s.c0 * SD, s.n);
            if (i + u >= to) key[u] = a.rows;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (key[u] >= a.rows) break; // padding, to the end
            if (key[u] != cur) {
                if (head) store_slot<A, V>(slot_at<A, V>(a, piece, SLOT_HEAD, v), acc);
                else add_to_grad<EG, V, TINY>(a, cur, s, acc);
                head = false;
                cur = key[u];
#pragma unroll
                for (int j = 0; j < V; j++) acc[j] = (A)0;
            }
            A x[V];
            d[u].unpack(x);
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] += x[j];
        }
    }
    if (head) store_slot<A, V>(slot_at<A, V>(a, piece, SLOT_HEAD, v), acc);
    else if (to < a.n && keys[to] == cur) store_slot<A, V>(slot_at<A, V>(a, piece, SLOT_TAIL, v), acc);
    else add_to_grad<EG, V, TINY>(a, cur, s, acc);
}

// One piece (of at most 64 tokens) and slab of 64 units by a wave.  Lane i holds token i's key and
// place, so that which token is the last of its row is one mask, and the rows' addresses are scalars.
// Eight tokens' rows are asked for at a time.  (Asking for what the finished rows hold together with them, instead of
// at the row's end, measured slower: 34-36 us against 31.4 for 16384 bf16 rows of 4 KiB into f32.)
template <int ED, int EG> DEV void sum_wide(const NboEmbedGradArgs &a, uint32_t wave)
{
    enum { V = Pair<ED, EG>::V, SD = sizeof(typename El<ED>::Bits), U = 8 };
    typedef typename El<EG>::A A;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t piece = wave / a.slabs, v = (wave - piece * a.slabs) * 64 + lane;
    if (piece >= a.pieces) return;
    const uint32_t from = piece * a.piece, len = a.n - from < a.piece ? a.n - from : a.piece;
    auto *keys = GLOBAL_PTR(const uint32_t, a.keys);
    const uint32_t at = from + (lane < len ? lane : len - 1);
    const uint32_t key = keys[at], pos = GLOBAL_PTR(const uint32_t, a.pos)[at];
    const uint32_t before = keys[from > 0 ? from - 1 : 0], behind = keys[from + len < a.n ? from + len : a.n - 1];
    const uint32_t cnt = (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(lane < len && key < a.rows)); // padding sorts last
    if (cnt == 0) return;
    const uint32_t next = __shfl_down(key, 1);
    const uint64_t ends = __builtin_amdgcn_ballot_w64(lane < cnt && (lane == cnt - 1 || key != next));
    bool head = from > 0 && before == (uint32_t)__builtin_amdgcn_readlane(key, 0);
    const bool tail = cnt == len && from + len < a.n && behind == (uint32_t)__builtin_amdgcn_readlane(key, len - 1);
    const bool on = v < a.units;
    const Span s = unit_span<V>(on ? v : a.units - 1, a.cols);
    A acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = (A)0;
    for (uint32_t i = 0; i < cnt; i += U) {
        Unit<ED, V> d[U];
#pragma unroll
        for (int u = 0; u < U; u++) { // (behind the last token: that one again)
            const uint32_t l = i + u < cnt ? i + u : cnt - 1;
            const char *row = (const char *)a.dy + __builtin_amdgcn_readlane(pos, l) * a.dy_stride;
            d[u].template load<false, true>(row + (uint64_t)s.c0 * SD, s.n);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i + u >= cnt) break;
            A x[V];
            d[u].unpack(x);
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] += x[j];
            if (!(ends >> (i + u) & 1)) continue;
            if (on) {
                if (head) store_slot<A, V>(slot_at<A, V>(a, piece, SLOT_HEAD, v), acc);
                else if (tail && i + u == cnt - 1) store_slot<A, V>(slot_at<A, V>(a, piece, SLOT_TAIL, v), acc);
                else add_to_grad<EG, V, false>(a, __builtin_amdgcn_readlane(key, i + u), s, acc);
            }
            head = false;
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] = (A)0;
        }
    }
}

// Zeros through the matrix from the front, one 16-byte store per thread and its wave is gone -- the shape in
// which this memory takes a fill fastest (6.6 TB/s over 1 GiB; waves that walk ranges of their own 5.0-5.8).
// `named`, if given, says which rows to leave alone.
DEV void clear_units(const NboClearArgs &c, const uint8_t *named, uint32_t wg)
{
    const uint64_t base = (uint64_t)wg * NBO_OPS_BLOCK;
    if (base + threadIdx.x >= c.u.total) return;
    UnitBase b = {};
    uint32_t on = 0, v = 0;
    if (named || !c.flat_bytes) {
        b = unit_base(c.u, base);
        unit_from(c.u, b, threadIdx.x, &on, &v);
    }
    if (named) {
        const uint32_t row = (uint32_t)b.row + on;
        if (GLOBAL_PTR(const uint8_t, named)[(row & ((1u << c.named_shift) - 1)) * c.named_range + (row >> c.named_shift)]) return;
    }
    if (c.flat_bytes) { // (few instructions per store; the last 16 bytes end with the matrix)
        const uint64_t o = (base + threadIdx.x) * 16;
        __builtin_nontemporal_store((u32x4_e)0, GLOBAL_PTR(u32x4_e, (char *)c.grad + (o + 16 <= c.flat_bytes ? o : c.flat_bytes - 16)));
        return;
    }
    const uint32_t bytes = (uint32_t)c.row_bytes;
    char *p = (char *)c.grad + b.row * c.grad_stride + on * c.grad_stride;
    if (bytes >= 16) { // (a row's last 16 bytes end with the row)
        __builtin_nontemporal_store((u32x4_e)0, GLOBAL_PTR(u32x4_e, p + (v * 16 + 16 <= bytes ? v * 16 : bytes - 16)));
    } else {
        for (uint32_t o = 0; o < bytes; o += 2) *GLOBAL_PTR(uint16_t, p + o) = 0;
    }
}

extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void nbo_embed_clear(const NboClearArgs c)
{
    clear_units(c, nullptr, folded_workgroup());
}

template <int ED, int EG, bool TINY> DEV void embed_sum_body(const NboEmbedGradArgs &a)
{
    const uint32_t wg = folded_workgroup();
    if (wg >= a.sum_wgs) {
        if (a.named) clear_units(a.clear, a.named, wg - a.sum_wgs);
        return;
    }
    const uint32_t wave = wg * (NBO_OPS_BLOCK / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (TINY || a.lanes < 64) sum_narrow<ED, EG, TINY>(a, wave);
    else sum_wide<ED, EG>(a, wave);
}

// Rows whose tokens span pieces.  A row that spans boundary k (between pieces k and k + 1) and begins in piece
// k is finished by that boundary's workgroups, one per slab of the row; a workgroup looks at a.edges boundaries.
// The row's sums are piece k's tail and the heads of the pieces behind, as many as begin with its key; the
// workgroup's waves -- groups of a.lanes lanes, where a row has few units -- take a run of them each.
// It waits for memory, one load after the other: 8192 tokens 5.6 us, 65536 13.  A row that has most of the tokens
// is one workgroup's per slab: 1024 sums of 2 KiB take 90 us, at the 23 GB/s that one compute unit reads -- more
// waves did not help (92 us with eight, 94 with sixteen), and cost every other row.
template <int ED, int EG, bool TINY> DEV void embed_join_body(const NboEmbedGradArgs &a)
{
    enum { V = Pair<ED, EG>::V, U = 8 };
    typedef typename El<EG>::A A;
    __shared__ A part[V][NBO_OPS_BLOCK];
    const uint32_t lane = threadIdx.x & 63u, group = threadIdx.x / a.lanes, groups = NBO_OPS_BLOCK / a.lanes;
    const uint32_t wg = folded_workgroup(), k0 = wg / a.slabs * a.edges;
    const uint32_t v = wg % a.slabs * 64 + threadIdx.x % a.lanes;
    const Span s = unit_span<V>(v < a.units ? v : a.units - 1, a.cols);
    auto *keys = GLOBAL_PTR(const uint32_t, a.keys);
    // lane j looks at boundary k0 + j, past the workgroup's own ones for where their rows end
    const uint32_t mine = k0 + lane;
    const bool edge = mine + 1 < a.pieces;
    const uint64_t at = edge ? (uint64_t)(mine + 1) * a.piece : a.piece; // (there are at least two pieces)
    const uint32_t key_at = keys[at], ahead = keys[at - 1], earlier = keys[at > a.piece ? at - a.piece - 1 : 0];
    uint64_t todo = __builtin_amdgcn_ballot_w64(edge && lane < a.edges && key_at < a.rows && ahead == key_at &&
                                                (mine == 0 || earlier != key_at));
    auto first_of = [&](uint64_t p) { return keys[(p < a.pieces ? p : a.pieces - 1) * a.piece]; };
    for (; todo; todo &= todo - 1) {
        const uint32_t j = __builtin_ctzll(todo), k = k0 + j, key = __builtin_amdgcn_readlane(key_at, j);
        Unit<EG, V> g;
        if (a.accumulate) g.template load<TINY, false>(grad_at<EG>(a, key, s), s.n);
        // the last piece that begins with this row (its boundary is inside the row): as far as the lanes have
        // looked, then, the order being sorted, among 64 evenly spaced pieces of what is left, as often as it takes
        const uint64_t same = __builtin_amdgcn_ballot_w64(edge && key_at == key) >> j; // (bit 0 is this boundary)
        const uint32_t seen = ~same ? (uint32_t)__builtin_ctzll(~same) : 64u;
        uint32_t last = k + seen;
        for (uint32_t end = j + seen < 64 ? last + 1 : a.pieces; end - last > 1;) {
            const uint32_t step = (end - last + 63) / 64;
            const uint64_t p = (uint64_t)last + (uint64_t)(lane + 1) * step;
            const uint32_t later = first_of(p);
            const uint64_t m = __builtin_amdgcn_ballot_w64(p < end && later == key); // (not all: p reaches end)
            const uint32_t c = (uint32_t)__builtin_ctzll(~m);
            last += c * step;
            if (end - last > step) end = last + step;
        }
        const uint32_t total = last - k, per = (total + groups - 1) / groups;
        A acc[V];
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] = (A)0;
        if (v < a.units) {
            if (group == 0) load_slot<A, V>(slot_at<A, V>(a, k, SLOT_TAIL, v), acc);
            const uint32_t lo = group * per, hi = lo + per < total ? lo + per : total;
            for (uint32_t i = lo; i < hi; i += U) {
                A x[U][V];
#pragma unroll
                for (int u = 0; u < U; u++) // (behind the run: its last one again)
                    load_slot<A, V>(slot_at<A, V>(a, k + 1 + (i + u < hi ? i + u : hi - 1), SLOT_HEAD, v), x[u]);
#pragma unroll
                for (int u = 0; u < U; u++) // (a select, no branch: into one the compiler would move the loads)
#pragma unroll
                    for (int j = 0; j < V; j++) acc[j] += i + u < hi ? x[u][j] : (A)0;
            }
        }
        __syncthreads(); // (the boundary before has been read)
#pragma unroll
        for (int j = 0; j < V; j++) part[j][threadIdx.x] = acc[j];
        __syncthreads();
        if (group == 0 && v < a.units) {
            for (uint32_t q = 1; q < groups; q++)
#pragma unroll
                for (int j = 0; j < V; j++) acc[j] += part[j][q * a.lanes + threadIdx.x];
            finish_row<EG, V>(a, key, s, g, acc);
        }
    }
}

// A few ids: one workgroup per token and slab of its row.  It reads all ids; unless an earlier token names
// the same row it adds up the rows of all tokens that do, each wave those in its run of the ids.  The
// workgroups behind clear the rows no token names.  One launch and three loads one after the other: 4.0 us for 96
// bf16 rows of 4 KiB.  Accumulating f32 rows of 3 KiB, 512 tokens take 6.6 us a call, 513 in three launches 14.1; all
// of one row, 9.9 and 12.4.
template <int ED, int EG, bool TINY> DEV void embed_direct_body(const NboEmbedGradArgs &a)
{
    enum { V = Pair<ED, EG>::V, SD = sizeof(typename El<ED>::Bits), WAVES = NBO_OPS_BLOCK / 64, U = 8 };
    enum { BLOCKS = NBO_EMBED_DIRECT_MAX / 64, RUN = BLOCKS / WAVES };
    typedef typename El<EG>::A A;
    __shared__ A part[WAVES][V][64];
    const uint32_t wg = folded_workgroup(), lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t key[BLOCKS] = {};
    if (a.n > 0) {
        uint64_t t[BLOCKS];
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) t[b] = b * 64 + lane < a.n ? b * 64 + lane : a.n - 1;
        load_keys<BLOCKS>(a.ids, a.ids64, t, a.rows, key);
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; b++)
        if (b * 64 + lane >= a.n) key[b] = 0xFFFFFFFFu;
    if (wg >= a.sum_wgs) {
        if (!a.clear.grad) return; // the unused end of a folded grid
        // a few rows to a wave
        const uint64_t from = ((uint64_t)(wg - a.sum_wgs) * WAVES + wave) * NBO_CLEAR_ROWS;
        if (from >= a.rows) return;
        const uint32_t count = a.rows - from < NBO_CLEAR_ROWS ? (uint32_t)(a.rows - from) : NBO_CLEAR_ROWS;
        uint64_t named = 0;
        for (uint32_t r = 0; r < count; r++) {
            uint64_t here = 0;
#pragma unroll
            for (int b = 0; b < BLOCKS; b++) here |= __builtin_amdgcn_ballot_w64(key[b] == (uint32_t)from + r);
            named |= (uint64_t)(here != 0) << r;
        }
        clear_rows(a.clear, from, count, named);
        return;
    }
    const uint32_t t = wg / a.slabs, v = (wg - t * a.slabs) * 64 + lane;
    uint32_t own = 0xFFFFFFFFu;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++)
        if (t / 64 == (uint32_t)b) own = __builtin_amdgcn_readlane(key[b], t & 63);
    if (own >= a.rows) return; // padding
    uint64_t mine[RUN] = {}; // this wave's tokens of the row
    bool first = true;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
        const uint64_t same = __builtin_amdgcn_ballot_w64(key[b] == own);
        if (t >= b * 64u && (same & (t - b * 64 >= 64 ? ~0ull : (1ull << (t - b * 64)) - 1))) first = false;
#pragma unroll
        for (int r = 0; r < RUN; r++)
            if ((uint32_t)b == wave * RUN + r) mine[r] = same;
    }
    if (!first) return;
    const Span s = unit_span<V>(v < a.units ? v : a.units - 1, a.cols);
    Unit<EG, V> g;
    if (a.accumulate) g.template load<TINY, false>(grad_at<EG>(a, own, s), s.n);
    A acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = (A)0;
#pragma unroll
    for (int r = 0; r < RUN; r++)
        for (uint64_t m = mine[r]; m;) {
            Unit<ED, V> d[U];
            uint32_t got = 0, i = 0;
#pragma unroll
            for (int u = 0; u < U; u++) { // (behind the last token: that one again)
                if (m) {
                    i = (wave * RUN + r) * 64 + __builtin_ctzll(m);
                    m &= m - 1;
                    got++;
                }
                d[u].template load<TINY, true>((const char *)a.dy + i * a.dy_stride + (uint64_t)s.c0 * SD, s.n);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if ((uint32_t)u >= got) break;
                A x[V];
                d[u].unpack(x);
#pragma unroll
                for (int j = 0; j < V; j++) acc[j] += x[j];
            }
        }
#pragma unroll
    for (int j = 0; j < V; j++) part[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; w++)
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] += part[w][j][lane];
    if (v < a.units) finish_row<EG, V>(a, own, s, g, acc);
}

#define NBO_EMBED_GRAD_KERNELS(suffix, ED, EG)                                                                   \
    extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void nbo_embed_sum_##suffix(const NboEmbedGradArgs a) \
    {                                                                                                            \
        if (a.cols >= (uint32_t)Pair<ED, EG>::V) embed_sum_body<ED, EG, false>(a);                               \
        else embed_sum_body<ED, EG, true>(a);                                                                     \
    }                                                                                                            \
    extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void nbo_embed_join_##suffix(const NboEmbedGradArgs a)\
    {                                                                                                            \
        if (a.cols >= (uint32_t)Pair<ED, EG>::V) embed_join_body<ED, EG, false>(a);                               \
        else embed_join_body<ED, EG, true>(a);                                                                     \
    }                                                                                                            \
    extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void nbo_embed_direct_##suffix(const NboEmbedGradArgs a) \
    {                                                                                                            \
        if (a.cols >= (uint32_t)Pair<ED, EG>::V) embed_direct_body<ED, EG, false>(a);                               \
        else embed_direct_body<ED, EG, true>(a);                                                                     \
    }
NBO_EMBED_GRAD_KERNELS(f32, NBO_F32, NBO_F32)
NBO_EMBED_GRAD_KERNELS(bf16, NBO_BF16, NBO_BF16)
NBO_EMBED_GRAD_KERNELS(f64, NBO_F64, NBO_F64)
NBO_EMBED_GRAD_KERNELS(f16, NBO_F16, NBO_F16)
NBO_EMBED_GRAD_KERNELS(bf16_f32, NBO_BF16, NBO_F32)
NBO_EMBED_GRAD_KERNELS(f16_f32, NBO_F16, NBO_F32)

// ---------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011): ten rounds of two 32 x 32 -> 64 bit products.  A block of eight elements costs some 100 instructions,
// which 16 bytes of bf16 hide: 32768 rows of 8 KiB 86.7 us, 6.2 TB/s of x and result.
DEV void philox(uint32_t block, uint32_t site, const NboRngDev &r, uint32_t (&w)[4])
{
    uint32_t c0 = block, c1 = site, c2 = (uint32_t)r.step, c3 = (uint32_t)(r.step >> 32);
    uint32_t k0 = (uint32_t)r.seed, k1 = (uint32_t)(r.seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
}

// One unit of V elements per thread.  PART: the last one of a row or the matrix, which has fewer.
template <int E, bool PART, bool ONCE> DEV void dropout_unit(const NboDropoutArgs &a, uint64_t row, uint64_t c, uint64_t e, uint32_t n)
{
    enum { V = Pair<E, E>::V, SZ = sizeof(typename El<E>::Bits) };
    typedef typename El<E>::A A;
    Unit<E, V> x, y;
    x.template load<PART, ONCE>((const char *)a.x + row * a.x_stride + c * SZ, n);
    if (a.residual) y.template load<PART, ONCE>((const char *)a.residual + row * a.residual_stride + c * SZ, n);
    const NboRngDev rng = *a.rng;
    uint32_t bits[V]; // each element's sixteen
    uint32_t w[4];
    const uint32_t sub = (uint32_t)e & 7u;
    philox((uint32_t)(e >> 3), a.site, rng, w);
    if (sub % V == 0) {
        // the unit's elements share one block of eight (all of it, or an aligned half or quarter)
        if (V == 8) {
#pragma unroll
            for (int j = 0; j < V; j++) bits[j] = j & 1 ? w[j >> 1 & 3] >> 16 : w[j >> 1 & 3] & 0xFFFFu;
        } else if (V == 4) {
            const uint32_t p = sub ? w[2] : w[0], q = sub ? w[3] : w[1];
#pragma unroll
            for (int j = 0; j < V; j++) bits[j] = (j & 1 ? (j < 2 ? p : q) >> 16 : (j < 2 ? p : q) & 0xFFFFu);
        } else {
            const uint32_t p = sub < 4 ? (sub < 2 ? w[0] : w[1]) : (sub < 6 ? w[2] : w[3]);
#pragma unroll
            for (int j = 0; j < V; j++) bits[j] = j & 1 ? p >> 16 : p & 0xFFFFu;
        }
    } else {
        // rows whose width is not a whole number of units: two blocks at most
        uint32_t w2[4];
        philox((uint32_t)((e + V - 1) >> 3), a.site, rng, w2);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const uint32_t q = sub + j; // < 16
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if ((q >> 1) == (uint32_t)i) word = w[i];
                if ((q >> 1) == (uint32_t)(i + 4)) word = w2[i];
            }
            bits[j] = q & 1 ? word >> 16 : word & 0xFFFFu;
        }
    }
    A f[V], g[V];
    x.unpack(f);
    const A scale = (A)a.scale;
#pragma unroll
    for (int j = 0; j < V; j++) f[j] = bits[j] >= a.thr ? f[j] * scale : (A)0;
    if (a.residual) {
        y.unpack(g);
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = g[j] + f[j];
    }
    x.pack(f);
    x.template store<ONCE>((char *)a.out + row * a.out_stride + c * SZ, 0, n);
}

template <int E> DEV void dropout_body(const NboDropoutArgs &a)
{
    enum { V = Pair<E, E>::V };
    const uint64_t base = (uint64_t)folded_workgroup() * NBO_OPS_BLOCK;
    const uint64_t unit = base + threadIdx.x;
    if (unit >= a.u.total) return;
    uint64_t row = 0, c = unit * V, e = c; // element `e` of the matrix, at column c of `row`
    uint32_t n;
    if (a.flat) {
        n = a.n - e < V ? (uint32_t)(a.n - e) : V;
    } else {
        uint32_t v;
        unit_at(a.u, unit_base(a.u, base), threadIdx.x, &row, &v);
        c = (uint64_t)v * V;
        e = row * a.cols + c;
        n = a.cols - c < V ? (uint32_t)(a.cols - c) : V;
    }
    if (n != V) dropout_unit<E, true, false>(a, row, c, e, n);
    else if (a.once) dropout_unit<E, false, true>(a, row, c, e, V);
    else dropout_unit<E, false, false>(a, row, c, e, V);
}

#define NBO_DROPOUT_KERNEL(name, E)                                                           \
    extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void name(const NboDropoutArgs a)  \
    {                                                                                         \
        dropout_body<E>(a);                                                                   \
    }
NBO_DROPOUT_KERNEL(nbo_dropout_f32, NBO_F32)
NBO_DROPOUT_KERNEL(nbo_dropout_bf16, NBO_BF16)
NBO_DROPOUT_KERNEL(nbo_dropout_f64, NBO_F64)
NBO_DROPOUT_KERNEL(nbo_dropout_f16, NBO_F16)

extern "C" __global__ void nbo_rng_advance(const NboRngAdvanceArgs a)
{
    if (threadIdx.x == 0) a.rng->step += a.steps;
}
