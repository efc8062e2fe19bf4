// gfx950 (CDNA4) kernels of the operators of include/nabla_ops.h: embedding lookup, its gradient,
// and dropout from a counter-based generator.  A code object of its own beside the optimizer's.
//
//   nbo_embed_*        out[t] = add[t] + scale * table[ids[t]]
//   nbo_order_rank     the ids in table order, by comparing all pairs (few ids)
//   nbo_order_hist / _scan / _scatter   ... by radix passes (many ids)
//   nbo_embed_sum_*    grad[v] (+)= scale * sum of the rows of dy that name v, in pieces of the order
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

// A unit of V elements of type E as it lies in memory: 16 bytes, or 32 where the other tensor of the
// operator has elements of half the size.
template <int E, int V> struct Unit {
    typedef typename El<E>::Bits Bits;
    typedef typename El<E>::A A;
    enum { SZ = sizeof(Bits), PER = 16 / SZ, N = V * SZ / 16 };
    u32x4 w[N];
    __device__ __forceinline__ void load(const char *p, uint32_t n) // n < V: a matrix narrower than a unit
    {
        if (n == V) {
#pragma unroll
            for (int k = 0; k < N; k++) w[k] = *GLOBAL_PTR(const u32x4_e, p + 16 * k);
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
    __device__ __forceinline__ void store(char *p, uint32_t skip, uint32_t n) const
    {
        if (skip == 0 && n == V) {
#pragma unroll
            for (int k = 0; k < N; k++) *GLOBAL_PTR(u32x4_e, p + 16 * k) = w[k];
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
DEV void unit_at(const NboUnits &u, const UnitBase &b, uint32_t x, uint64_t *row, uint32_t *v)
{
    const uint32_t y = b.first + x;
    uint32_t q;
    if (u.per_row == 1) q = y;
    else if (u.per_row < 1024) q = __umulhi(y, u.m32);
    else q = y >= u.per_row ? 1u : 0u;
    *row = b.row + q;
    *v = y - q * u.per_row;
}

// the id of token t as a row of the table, or `rows` for an id outside it
DEV uint32_t load_key(const void *ids, uint32_t ids64, uint64_t t, uint32_t rows)
{
    if (ids64) {
        const uint64_t id = GLOBAL_PTR(const uint64_t, ids)[t];
        return id < rows ? (uint32_t)id : rows;
    }
    const uint32_t id = GLOBAL_PTR(const uint32_t, ids)[t];
    return id < rows ? id : rows;
}

// ---------------------------------------------------------------------------------
// The lookup: U units per thread, all ids read, then all rows, then all stores.
template <int ET, int EO, int U> DEV void embed_body(const NboEmbedArgs &a)
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
        unit_at(a.u, b, x, &t[k], &v[k]);
        key[k] = on[k] ? load_key(a.ids, a.ids64, t[k], a.rows) : a.rows;
    }
    Unit<ET, V> row[U];
    Unit<EO, V> add[U];
#pragma unroll
    for (int k = 0; k < U; k++) {
        const Span s = unit_span<V>(v[k], a.cols);
        row[k].clear();
        if (key[k] < a.rows) row[k].load((const char *)a.table + key[k] * a.table_stride + (uint64_t)s.c0 * ST, s.n);
        if (a.add && on[k]) add[k].load((const char *)a.add + t[k] * a.add_stride + (uint64_t)s.c0 * SO, s.n);
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
        o.store((char *)a.out + t[k] * a.out_stride + (uint64_t)s.c0 * SO, s.skip, s.n);
    }
}

#define NBO_EMBED_KERNEL(name, ET, EO)                                                      \
    extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void name(const NboEmbedArgs a)  \
    {                                                                                       \
        embed_body<ET, EO, 1>(a);                                                           \
    }
NBO_EMBED_KERNEL(nbo_embed_f32, NBO_F32, NBO_F32)
NBO_EMBED_KERNEL(nbo_embed_bf16, NBO_BF16, NBO_BF16)
NBO_EMBED_KERNEL(nbo_embed_f64, NBO_F64, NBO_F64)
NBO_EMBED_KERNEL(nbo_embed_f16, NBO_F16, NBO_F16)
NBO_EMBED_KERNEL(nbo_embed_f32_bf16, NBO_F32, NBO_BF16)
NBO_EMBED_KERNEL(nbo_embed_f32_f16, NBO_F32, NBO_F16)

// ---------------------------------------------------------------------------------
// Table order by all pairs: a token's place is the number of (key, token) pairs before its own.
// One workgroup ranks 64 tokens, one per lane; its sixteen waves share the ids, which lie in LDS.
extern "C" __global__ __launch_bounds__(NBO_RANK_BLOCK) void nbo_order_rank(const NboOrderArgs a)
{
    enum { WAVES = NBO_RANK_BLOCK / 64 };
    __shared__ uint32_t keys[NBO_RANK_MAX];
    __shared__ uint32_t before[WAVES][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t blocks = (a.n + 63) / 64; // of 64 keys; the last is filled up with keys that are before none
    for (uint32_t i = threadIdx.x; i < blocks * 64; i += NBO_RANK_BLOCK)
        keys[i] = i < a.n ? load_key(a.ids, a.ids64, i, a.rows) : 0xFFFFFFFFu;
    __syncthreads();
    const uint32_t own = blockIdx.x, mine = keys[own * 64 + lane];
    const uint32_t per = (blocks + WAVES - 1) / WAVES;
    const uint32_t lo = wave * per, hi = lo + per < blocks ? lo + per : blocks;
    uint32_t cnt = 0;
    for (uint32_t blk = lo; blk < hi; blk++) {
        const u32x4 *k4 = (const u32x4 *)(keys + blk * 64);
        if (blk == own) {
            for (uint32_t j = 0; j < 64; j++) {
                const uint32_t k = keys[blk * 64 + j];
                cnt += k < mine || (k == mine && j < lane);
            }
        } else {
            // equal keys of earlier blocks are before this one's, of later blocks behind
            const uint32_t bound = blk < own ? mine + 1 : mine;
#pragma unroll 4
            for (uint32_t j = 0; j < 16; j++) {
                const u32x4 k = k4[j];
                cnt += k.x < bound;
                cnt += k.y < bound;
                cnt += k.z < bound;
                cnt += k.w < bound;
            }
        }
    }
    before[wave][lane] = cnt;
    __syncthreads();
    const uint32_t t = own * 64 + lane;
    if (wave == 0 && t < a.n) {
        uint32_t rank = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) rank += before[w][lane];
        GLOBAL_PTR(uint32_t, a.keys_out)[rank] = mine;
        GLOBAL_PTR(uint32_t, a.pos_out)[rank] = t;
    }
}

// ---------------------------------------------------------------------------------
// Table order by stable radix passes of up to ten bits, least significant first.  Per pass: how often
// each digit occurs in each tile; the running sums over the tiles, per digit; every id to its place.
DEV uint32_t order_key(const NboOrderArgs &a, uint32_t i)
{
    return a.keys_in ? GLOBAL_PTR(const uint32_t, a.keys_in)[i] : load_key(a.ids, a.ids64, i, a.rows);
}

extern "C" __global__ __launch_bounds__(NBO_RADIX_BLOCK) void nbo_order_hist(const NboOrderArgs a)
{
    __shared__ uint32_t count[1u << NBO_RADIX_BITS];
    for (uint32_t d = threadIdx.x; d < a.digits; d += NBO_RADIX_BLOCK) count[d] = 0;
    __syncthreads();
    const uint32_t first = blockIdx.x * NBO_RADIX_TILE;
#pragma unroll
    for (uint32_t k = 0; k < NBO_RADIX_TILE / NBO_RADIX_BLOCK; k++) {
        const uint32_t i = first + k * NBO_RADIX_BLOCK + threadIdx.x;
        // (counts: the order of these additions changes nothing)
        if (i < a.n) atomicAdd(&count[(order_key(a, i) >> a.shift) & (a.digits - 1)], 1u);
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < a.digits; d += NBO_RADIX_BLOCK)
        GLOBAL_PTR(uint32_t, a.hist)[(uint64_t)d * a.tiles + blockIdx.x] = count[d];
}

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

extern "C" __global__ __launch_bounds__(NBO_RADIX_BLOCK) void nbo_order_scatter(const NboOrderArgs a)
{
    enum { WAVES = NBO_RADIX_BLOCK / 64, ROWS = NBO_RADIX_TILE / NBO_RADIX_BLOCK };
    __shared__ uint32_t count[WAVES][1u << NBO_RADIX_BITS]; // per wave, then: where the wave's next one goes
    __shared__ uint32_t wsum[WAVES];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t d = threadIdx.x; d < a.digits; d += NBO_RADIX_BLOCK)
#pragma unroll
        for (int w = 0; w < WAVES; w++) count[w][d] = 0;
    // each wave takes a run of the tile, in order, 64 ids at a time
    const uint32_t first = blockIdx.x * NBO_RADIX_TILE + wave * (ROWS * 64) + lane;
    uint32_t key[ROWS], pos[ROWS], rank[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const uint32_t i = first + r * 64;
        key[r] = i < a.n ? order_key(a, i) : 0;
        pos[r] = i < a.n ? (a.pos_in ? GLOBAL_PTR(const uint32_t, a.pos_in)[i] : i) : 0;
    }
    __syncthreads();
    volatile uint32_t *mine = count[wave];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const bool on = first + r * 64 < a.n;
        const uint32_t d = (key[r] >> a.shift) & (a.digits - 1);
        uint64_t same = __builtin_amdgcn_ballot_w64(on);
        for (uint32_t bit = 1; bit < a.digits; bit <<= 1) { // lanes with the same digit
            const uint64_t m = __builtin_amdgcn_ballot_w64((d & bit) != 0);
            same &= (d & bit) ? m : ~m;
        }
        const uint32_t ahead = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
        uint32_t seen = 0;
        if (on) seen = mine[d];
        rank[r] = seen + ahead;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (on && ahead == 0) mine[d] = seen + (uint32_t)__popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // where each digit starts: the digits below it, the tiles before this one, the waves before each
    const uint32_t per = (a.digits + NBO_RADIX_BLOCK - 1) / NBO_RADIX_BLOCK; // at most 2
    uint32_t tot[2] = {0, 0};
    for (uint32_t k = 0; k < per; k++) {
        const uint32_t d = threadIdx.x * per + k;
        if (d < a.digits) tot[k] = GLOBAL_PTR(const uint32_t, a.totals)[d];
    }
    const uint32_t up = wave_scan(tot[0] + tot[1]);
    if (lane == 63) wsum[wave] = up;
    __syncthreads();
    uint32_t below = up - (tot[0] + tot[1]);
    for (uint32_t w = 0; w < wave; w++) below += wsum[w];
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
        if (first + r * 64 < a.n) {
            const uint32_t at = count[wave][(key[r] >> a.shift) & (a.digits - 1)] + rank[r];
            GLOBAL_PTR(uint32_t, a.keys_out)[at] = key[r];
            GLOBAL_PTR(uint32_t, a.pos_out)[at] = pos[r];
        }
}

// ---------------------------------------------------------------------------------
// The sums.  The order is cut into pieces of a.piece tokens; `lanes` lanes, one unit of the row each,
// walk a piece and add up the rows of dy.  A row of the table all of whose tokens lie in the piece is
// finished there; the sums of one that began in an earlier piece or goes on into the next are left in
// the piece's two slots, for the join.  So a row that half the batch names is added up by many
// waves, and in the same order of additions on every run.
template <int EG, int V> DEV void add_to_grad(const NboEmbedGradArgs &a, uint32_t key, const Span &s,
                                              typename El<EG>::A (&x)[V])
{
    typedef typename El<EG>::A A;
    char *p = (char *)a.grad + key * a.grad_stride + (uint64_t)s.c0 * sizeof(typename El<EG>::Bits);
    const A scale = (A)a.scale;
    Unit<EG, V> g;
    if (a.accumulate) {
        A y[V];
        g.load(p, s.n);
        g.unpack(y);
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = y[j] + scale * x[j];
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = scale * x[j];
    }
    g.pack(x);
    g.store(p, s.skip, s.n);
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

// first place in keys[lo .. hi) whose key is not below `key`
DEV uint32_t lower_bound(const uint32_t *keys, uint32_t lo, uint32_t hi, uint32_t key)
{
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (GLOBAL_PTR(const uint32_t, keys)[mid] < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}
// ... by a whole wave, 64 places at a time
DEV uint32_t lower_bound_wave(const uint32_t *keys, uint32_t n, uint32_t key)
{
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t lo = 0, len = n; // the place is in [lo, lo + len]
    while (len > 0) {
        const uint32_t step = (len + 63) / 64;
        const uint64_t i = (uint64_t)lo + (uint64_t)lane * step;
        const bool below = lane * (uint64_t)step < len && GLOBAL_PTR(const uint32_t, keys)[i] < key;
        const uint32_t c = (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(below)); // probes 0 .. c - 1 are below
        if (c == 0) return lo;
        const uint32_t from = (c - 1) * step + 1; // behind the last probe that is below
        const uint32_t to = c * step < len ? c * step : len;
        lo += from;
        len = to > from ? to - from : 0;
    }
    return lo;
}

// Zeros in the rows from..from + 63 at most whose bit in `named` is not set, by the whole workgroup.
DEV void clear_rows(const NboEmbedGradArgs &a, uint32_t from, uint32_t count, uint64_t named)
{
    for (uint32_t r = 0; r < count; r++) {
        if (named >> r & 1) continue;
        char *p = (char *)a.grad + (uint64_t)(from + r) * a.grad_stride;
        const u32x4 z = 0;
        const uint64_t nvec = a.row_bytes / 16;
        for (uint64_t i = threadIdx.x; i < nvec; i += NBO_OPS_BLOCK) *GLOBAL_PTR(u32x4_e, p + i * 16) = z;
        // what is left is less than a vector: whole elements, two bytes at a time
        const uint32_t left = (uint32_t)(a.row_bytes - nvec * 16) / 2;
        if (threadIdx.x < left) *GLOBAL_PTR(uint16_t, p + nvec * 16 + threadIdx.x * 2) = 0;
    }
}

DEV void clear_unnamed(const NboEmbedGradArgs &a, uint32_t wg)
{
    __shared__ uint64_t named;
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t from = (uint64_t)wg * a.zero_rows;
    if (from >= a.rows) return;
    const uint32_t count = a.rows - from < a.zero_rows ? (uint32_t)(a.rows - from) : a.zero_rows;
    if (threadIdx.x < 64) {
        const uint32_t lo = lower_bound_wave(a.keys, a.n, (uint32_t)from);
        const uint32_t hi = lower_bound_wave(a.keys, a.n, (uint32_t)from + count);
        bool here = false;
        if (lo < hi && lane < count) {
            const uint32_t at = lower_bound(a.keys, lo, hi, (uint32_t)from + lane);
            here = at < hi && GLOBAL_PTR(const uint32_t, a.keys)[at] == (uint32_t)from + lane;
        }
        const uint64_t m = __builtin_amdgcn_ballot_w64(here);
        if (lane == 0) named = m;
    }
    __syncthreads();
    clear_rows(a, (uint32_t)from, count, named);
}

template <int ED, int EG> DEV void embed_sum_body(const NboEmbedGradArgs &a)
{
    enum { V = Pair<ED, EG>::V, SD = sizeof(typename El<ED>::Bits), U = 8 };
    typedef typename El<EG>::A A;
    const uint32_t wg = folded_workgroup();
    if (wg >= a.sum_wgs) {
        if (wg - a.sum_wgs < a.zero_wgs) clear_unnamed(a, wg - a.sum_wgs);
        return;
    }
    const uint32_t wave = wg * (NBO_OPS_BLOCK / 64) + threadIdx.x / 64, lane = threadIdx.x & 63u;
    uint32_t piece, v;
    if (a.lanes == 64) {
        piece = wave / a.slabs;
        v = (wave - piece * a.slabs) * 64 + lane;
    } else {
        piece = wave * (64 / a.lanes) + lane / a.lanes;
        v = lane % a.lanes;
    }
    if (piece >= a.pieces || v >= a.units) return;
    const Span s = unit_span<V>(v, a.cols);
    const uint32_t from = piece * a.piece, to = a.n - from < a.piece ? a.n : from + a.piece;
    auto *keys = GLOBAL_PTR(const uint32_t, a.keys);
    auto *pos = GLOBAL_PTR(const uint32_t, a.pos);
    uint32_t cur = keys[from];
    bool head = from > 0 && keys[from - 1] == cur;
    A acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = (A)0;
    for (uint32_t i = from; i < to; i++) {
        const uint32_t key = keys[i];
        if (key >= a.rows) break; // padding, to the end
        if (key != cur) {
            if (head) store_slot<A, V>(slot_at<A, V>(a, piece, SLOT_HEAD, v), acc);
            else add_to_grad<EG, V>(a, cur, s, acc);
            head = false;
            cur = key;
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] = (A)0;
        }
        Unit<ED, V> d;
        A x[V];
        d.load((const char *)a.dy + pos[i] * a.dy_stride + (uint64_t)s.c0 * SD, s.n);
        d.unpack(x);
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] += x[j];
    }
    if (cur >= a.rows) return; // nothing but padding
    if (head) store_slot<A, V>(slot_at<A, V>(a, piece, SLOT_HEAD, v), acc);
    else if (to < a.n && keys[to] == cur) store_slot<A, V>(slot_at<A, V>(a, piece, SLOT_TAIL, v), acc);
    else add_to_grad<EG, V>(a, cur, s, acc);
}

// Rows whose tokens span pieces: the workgroups of boundary k (between pieces k and k + 1), one per slab
// of the row, finish the row that spans it and begins in piece k.  Its sums are piece k's tail and the
// heads of the pieces behind, as many as begin with its key; the four waves take a run of them each.
template <int ED, int EG> DEV void embed_join_body(const NboEmbedGradArgs &a)
{
    enum { V = Pair<ED, EG>::V, WAVES = NBO_OPS_BLOCK / 64 };
    typedef typename El<EG>::A A;
    __shared__ A part[WAVES][V][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t slabs = (a.units + 63) / 64;
    const uint32_t wg = folded_workgroup(), k = wg / slabs, v = (wg - k * slabs) * 64 + lane;
    if (k + 1 >= a.pieces) return;
    auto *keys = GLOBAL_PTR(const uint32_t, a.keys);
    const uint64_t edge = (uint64_t)(k + 1) * a.piece;
    const uint32_t key = keys[edge];
    if (key >= a.rows || keys[edge - 1] != key) return; // no row spans this boundary
    if (k > 0 && keys[edge - a.piece - 1] == key) return; // ... or it began earlier
    uint32_t last = k + 1; // the last piece that begins with this row (its boundary is inside the row)
    for (;;) {
        const uint64_t p = (uint64_t)last + 1 + lane;
        const bool more = p < a.pieces && keys[p * a.piece] == key;
        const uint64_t m = ~__builtin_amdgcn_ballot_w64(more);
        const uint32_t c = m ? (uint32_t)__builtin_ctzll(m) : 64u;
        last += c;
        if (c < 64) break;
    }
    const uint32_t total = last - k, per = (total + WAVES - 1) / WAVES;
    A acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = (A)0;
    if (v < a.units) {
        if (wave == 0) load_slot<A, V>(slot_at<A, V>(a, k, SLOT_TAIL, v), acc);
        const uint32_t lo = wave * per, hi = lo + per < total ? lo + per : total;
        for (uint32_t i = lo; i < hi; i++) {
            A x[V];
            load_slot<A, V>(slot_at<A, V>(a, k + 1 + i, SLOT_HEAD, v), x);
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] += x[j];
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) part[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave == 0 && v < a.units) {
#pragma unroll
        for (int w = 1; w < WAVES; w++)
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] += part[w][j][lane];
        const Span s = unit_span<V>(v, a.cols);
        add_to_grad<EG, V>(a, key, s, acc);
    }
}

// A few ids: one wave per token and slab.  It reads all ids; unless an earlier token names the same
// row it adds up the rows of all tokens that do.  The workgroups behind clear the other rows.
template <int ED, int EG> DEV void embed_direct_body(const NboEmbedGradArgs &a)
{
    enum { V = Pair<ED, EG>::V, SD = sizeof(typename El<ED>::Bits), BLOCKS = NBO_EMBED_DIRECT_MAX / 64 };
    typedef typename El<EG>::A A;
    const uint32_t wg = folded_workgroup(), lane = threadIdx.x & 63u;
    uint32_t key[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
        const uint32_t i = b * 64 + lane;
        key[b] = i < a.n ? load_key(a.ids, a.ids64, i, a.rows) : 0xFFFFFFFFu;
    }
    if (wg >= a.sum_wgs) {
        const uint64_t from = (uint64_t)(wg - a.sum_wgs) * a.zero_rows;
        if (wg - a.sum_wgs >= a.zero_wgs || from >= a.rows) return;
        const uint32_t count = a.rows - from < a.zero_rows ? (uint32_t)(a.rows - from) : a.zero_rows;
        uint32_t lo = 0, hi = 0; // bit r: row from + r is named
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            const uint64_t r = (uint64_t)key[b] - from;
            if (key[b] >= from && r < count) (r < 32 ? lo : hi) |= 1u << (r & 31);
        }
#pragma unroll
        for (int s = 1; s < 64; s *= 2) {
            lo |= __shfl_xor(lo, s);
            hi |= __shfl_xor(hi, s);
        }
        clear_rows(a, (uint32_t)from, count, (uint64_t)hi << 32 | lo);
        return;
    }
    const uint32_t wave = wg * (NBO_OPS_BLOCK / 64) + threadIdx.x / 64;
    const uint32_t t = wave / a.slabs, v = (wave - t * a.slabs) * 64 + lane;
    if (t >= a.n) return;
    uint32_t own = 0xFFFFFFFFu;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++)
        if (t / 64 == (uint32_t)b) own = __shfl(key[b], t & 63);
    if (own >= a.rows) return; // padding
    uint64_t same[BLOCKS];
    bool first = true;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
        same[b] = __builtin_amdgcn_ballot_w64(key[b] == own);
        if (t >= b * 64u && (same[b] & (t - b * 64 >= 64 ? ~0ull : (1ull << (t - b * 64)) - 1))) first = false;
    }
    if (!first || v >= a.units) return;
    const Span s = unit_span<V>(v, a.cols);
    A acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = (A)0;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++)
        for (uint64_t m = same[b]; m; m &= m - 1) {
            const uint64_t i = b * 64 + __builtin_ctzll(m);
            Unit<ED, V> d;
            A x[V];
            d.load((const char *)a.dy + i * a.dy_stride + (uint64_t)s.c0 * SD, s.n);
            d.unpack(x);
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] += x[j];
        }
    add_to_grad<EG, V>(a, own, s, acc);
}

#define NBO_EMBED_GRAD_KERNELS(suffix, ED, EG)                                                                   \
    extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void nbo_embed_sum_##suffix(const NboEmbedGradArgs a) \
    {                                                                                                            \
        embed_sum_body<ED, EG>(a);                                                                               \
    }                                                                                                            \
    extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void nbo_embed_join_##suffix(const NboEmbedGradArgs a)\
    {                                                                                                            \
        embed_join_body<ED, EG>(a);                                                                              \
    }                                                                                                            \
    extern "C" __global__ __launch_bounds__(NBO_OPS_BLOCK) void nbo_embed_direct_##suffix(const NboEmbedGradArgs a) \
    {                                                                                                            \
        embed_direct_body<ED, EG>(a);                                                                            \
    }
NBO_EMBED_GRAD_KERNELS(f32, NBO_F32, NBO_F32)
NBO_EMBED_GRAD_KERNELS(bf16, NBO_BF16, NBO_BF16)
NBO_EMBED_GRAD_KERNELS(f64, NBO_F64, NBO_F64)
NBO_EMBED_GRAD_KERNELS(f16, NBO_F16, NBO_F16)
NBO_EMBED_GRAD_KERNELS(bf16_f32, NBO_BF16, NBO_F32)
NBO_EMBED_GRAD_KERNELS(f16_f32, NBO_F16, NBO_F32)

// ---------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011): ten rounds of two 32 x 32 -> 64 bit products.
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

template <int E> DEV void dropout_body(const NboDropoutArgs &a)
{
    enum { V = Pair<E, E>::V, SZ = sizeof(typename El<E>::Bits) };
    typedef typename El<E>::A A;
    const uint64_t base = (uint64_t)folded_workgroup() * NBO_OPS_BLOCK;
    const uint64_t unit = base + threadIdx.x;
    if (unit >= a.u.total) return;
    uint64_t row = 0, c = unit * V, e = c; // element `e` of the matrix, at column c of `row`
    Span s = {0, 0, V};
    if (a.flat) {
        s.n = a.n - e < V ? (uint32_t)(a.n - e) : V;
    } else {
        uint32_t v;
        unit_at(a.u, unit_base(a.u, base), threadIdx.x, &row, &v);
        c = (uint64_t)v * V;
        e = row * a.cols + c;
        s.n = a.cols - c < V ? (uint32_t)(a.cols - c) : V;
    }
    Unit<E, V> x, y;
    x.load((const char *)a.x + row * a.x_stride + c * SZ, s.n);
    if (a.residual) y.load((const char *)a.residual + row * a.residual_stride + c * SZ, s.n);
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
    x.store((char *)a.out + row * a.out_stride + c * SZ, 0, s.n);
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
