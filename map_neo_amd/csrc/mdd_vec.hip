// Document vectors: embedding lookup and its gradient, root-mean-square norm (plain, to 8 bits, backward), cosines of
// candidate edges on 8-bit rows, edge ordering.  Declarations and contracts: include/mdd.h.
#include "mdd_vec.h"

#include <type_traits>
#include <utility>

using namespace mddi;

namespace {

constexpr uint32_t NO_ROW = 0xFFFFFFFFu;

// ------------------------------------------------------------------------------------------------ embedding lookup
// out[d] = f_d * sum of table rows.  A wave sums one document: `lpr` lanes side by side cover a row's columns (8 each; with NS = 2
// all 64 lanes take 8 in either half of 1024, and wider rows are shared by waves of their own), the 64 / lpr lane groups take
// neighbouring positions.  64 ids are read at once, a batch ahead; those that name a row move up to the lowest lanes, so that
// padding costs nothing behind this point, and are handed out by lane, up to eight rows per group in flight.
// The table of a static embedding (64000 x 256 in bf16: 33 MB) lives in the last-level cache, so the kernel is bound by
// the caches' gather rate, not by HBM: 40000 documents of 480 ids, 9.7 GB of rows, take 480 us = 20 TB/s; a third of the lines
// miss L2, and from a table that fits there the same sums take 330 us.  Sixteen rows in flight cost more in resident waves than
// they gain (690 us), four are as good as eight.
//
// Documents longer than a piece (2^piece_log2 ids) would leave one wave with all the work: the id axis is cut into pieces, a
// piece's share of a long document goes to a workspace row in float, and pool_join_kernel adds the shares in order.  A piece
// holds at most two shares -- of the document it starts in (slot 0) and of the one it ends in (slot 1) -- because a
// document strictly inside a piece is not long.
struct PoolArgs {
    const void* table;
    uint64_t n_rows;
    uint32_t row_bytes;  // from a table row to the next
    uint32_t dim, lpr;
    uint32_t slabs;  // of 256 columns, shared out by block (column_slabs); 1: all columns
    const void* ids;
    int id_bytes;
    uint64_t n_ids;
    const uint64_t* offsets;
    uint64_t n_docs;
    int mean;
    float scale;
    const uint32_t* row_count;  // gradient of a mean: ids of the document a row stands for; its rows weigh scale / count
    uint32_t piece_log2;
    uint64_t n_pieces;
    float* part;       // [piece][slot][dim]
    uint32_t* part_n;  // [piece][slot] ids that name a row
    uint64_t* begins;  // [piece] the long document that begins in it, ~0 without one
    void* out;
};

// row that position p's id names, or NO_ROW (negative ids become huge: padding as well)
__device__ __forceinline__ uint32_t named_row(const void* ids, int id_bytes, uint64_t p, uint64_t n_rows) {
    const uint64_t id = id_bytes == 4 ? (uint64_t)(int64_t)reinterpret_cast<const int32_t*>(ids)[p] : (uint64_t)reinterpret_cast<const int64_t*>(ids)[p];
    return id < n_rows ? (uint32_t)id : NO_ROW;
}

//
// A lane's eight columns never reach over the row's end: the last lane starts early enough, and where that makes it overlap its
// neighbour both compute and store the same numbers.  So every access is one of eight elements, without a branch.  Rows
// narrower than that (NARROW) take a path of single elements.
template <bool NARROW>
__device__ __forceinline__ uint32_t lane_col(uint32_t col, uint32_t dim) {
    return NARROW ? 0 : col < dim - 8 ? col : dim - 8;
}
template <typename T, bool NARROW, bool ONCE = false>
__device__ __forceinline__ typename vec8<T>::raw load_cols(const T* __restrict__ p, uint32_t dim) {
    if constexpr (ONCE && !NARROW) return __builtin_nontemporal_load(reinterpret_cast<const typename vec8<T>::raw_any*>(p));
    else return load8_raw<T>(p, NARROW ? dim : 8);
}

// U rows per lane group, held by the lanes from byte lane index `first` on in steps of `step`.  ALL: every one of them is
// named; otherwise NO_ROW is among them, for which row 0 is read and dropped, whatever it holds, NaN included.
template <typename T, int NS, bool WEIGHTED, bool NARROW, bool ONCE, bool ALL, int U>
__device__ __forceinline__ void add_rows(const PoolArgs& a, const T* __restrict__ (&table)[NS], uint32_t held, float weight, int first, int step, f32x8 (&acc)[NS]) {
    typename vec8<T>::raw raw[U][NS];
    uint32_t at[U];
#pragma unroll
    for (int u = 0; u < U; u++) at[u] = (uint32_t)__builtin_amdgcn_ds_bpermute(first + u * step, (int)held);
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint64_t off = (uint64_t)(ALL || at[u] != NO_ROW ? at[u] : 0) * a.row_bytes;
#pragma unroll
        for (int n = 0; n < NS; n++) raw[u][n] = load_cols<T, NARROW, ONCE>(reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(table[n]) + off), a.dim);
    }
    __builtin_amdgcn_sched_barrier(0);  // all loads first: left alone, the compiler takes them one by one to save registers
    if constexpr (std::is_same_v<T, __bf16> && !WEIGHTED && ALL && !NARROW && U >= 2) {
        // Two rows at once: their elements of a column side by side, times one and one, added to the sum -- an instruction per
        // element where a conversion and an addition are two.  The sum has at most the error of two additions, subnormal numbers
        // included (its form for fp16 drops those and is not used).  40000 documents of 480 x 256: 516 -> 488 us.
        typedef __bf16 two __attribute__((ext_vector_type(2)));
        const two ones = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
        for (int u = 0; u < U; u += 2)
#pragma unroll
            for (int n = 0; n < NS; n++) {
                const u32x4 x = __builtin_bit_cast(u32x4, raw[u][n]), y = __builtin_bit_cast(u32x4, raw[u + 1][n]);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    acc[n][2 * k] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(two, __builtin_amdgcn_perm(y[k], x[k], 0x05040100u)), ones, acc[n][2 * k], false);
                    acc[n][2 * k + 1] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(two, __builtin_amdgcn_perm(y[k], x[k], 0x07060302u)), ones, acc[n][2 * k + 1], false);
                }
            }
        return;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const float w = WEIGHTED ? __int_as_float(__builtin_amdgcn_ds_bpermute(first + u * step, __float_as_int(weight))) : 1.0f;
#pragma unroll
        for (int n = 0; n < NS; n++) {
            f32x8 v = __builtin_convertvector(raw[u][n], f32x8);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float x = ALL || at[u] != NO_ROW ? v[k] : 0.0f;
                acc[n][k] = WEIGHTED ? fmaf(x, w, acc[n][k]) : acc[n][k] + x;
            }
        }
    }
}

// sum of the rows named by ids [beg, end) in this lane's columns; n_named = ids that name a row.  Call with all lanes.
template <typename T, int NS, bool WEIGHTED, bool NARROW, bool ONCE>
__device__ __forceinline__ void sum_span(const PoolArgs& a, uint64_t beg, uint64_t end, const uint32_t (&col)[NS], f32x8 (&acc)[NS], uint32_t& n_named) {
    const int lane = (int)lane_id(), lpr = NS == 2 ? 64 : (int)a.lpr, G = 64 / lpr, g = lane / lpr;
    const T* __restrict__ table[NS];
#pragma unroll
    for (int n = 0; n < NS; n++) {
        table[n] = reinterpret_cast<const T*>(a.table) + col[n];
        acc[n] = 0.0f;
    }
    n_named = 0;
    uint32_t row = beg + lane < end ? named_row(a.ids, a.id_bytes, beg + lane, a.n_rows) : NO_ROW;
    for (uint64_t p = beg; p < end; p += 64) {
        const uint32_t next = p + 64 + lane < end ? named_row(a.ids, a.id_bytes, p + 64 + lane, a.n_rows) : NO_ROW;
        const uint64_t named = __ballot(row != NO_ROW);
        const int n = __popcll(named);
        n_named += (uint32_t)n;
        float w = 0.0f;
        if (WEIGHTED && row != NO_ROW) w = a.scale / (float)a.row_count[row];
        if (n < 64) {  // named lanes to 0 .. n - 1 in their order, the others behind them
            const uint32_t up = below(named), to = row != NO_ROW ? up : n + lane - up;
            row = (uint32_t)__builtin_amdgcn_ds_permute((int)to * 4, (int)row);
            if (WEIGHTED) w = __int_as_float(__builtin_amdgcn_ds_permute((int)to * 4, __float_as_int(w)));
        }
        // steps of G rows, one per group: eight at a time, what is left in batches of 4, 2, 1 (at most three more round trips,
        // no row read twice), and last the groups that get one row more than the others
        const int steps = n >> __builtin_ctz(G);
        int j = 0;
        if constexpr (!NARROW) {
            for (; j + 8 <= steps; j += 8) add_rows<T, NS, WEIGHTED, NARROW, ONCE, true, 8>(a, table, row, w, (j * G + g) * 4, G * 4, acc);
            if (j + 4 <= steps) add_rows<T, NS, WEIGHTED, NARROW, ONCE, true, 4>(a, table, row, w, (j * G + g) * 4, G * 4, acc), j += 4;
            if (j + 2 <= steps) add_rows<T, NS, WEIGHTED, NARROW, ONCE, true, 2>(a, table, row, w, (j * G + g) * 4, G * 4, acc), j += 2;
        }
        for (; j < steps; j++) add_rows<T, NS, WEIGHTED, NARROW, ONCE, true, 1>(a, table, row, w, (j * G + g) * 4, G * 4, acc);
        if (j * G < n) add_rows<T, NS, WEIGHTED, NARROW, ONCE, false, 1>(a, table, row, w, (j * G + g) * 4, G * 4, acc);
        row = next;
    }
    for (int m = lpr; m < 64; m <<= 1)
#pragma unroll
        for (int n = 0; n < NS; n++)
#pragma unroll
            for (int k = 0; k < 8; k++) acc[n][k] += __shfl_xor(acc[n][k], m, 64);
}

__device__ __forceinline__ float pool_factor(const PoolArgs& a, uint32_t n_named) {
    if (a.row_count) return 1.0f;  // the rows carried their weights
    return a.mean ? (n_named ? a.scale / (float)n_named : 0.0f) : a.scale;
}

// last document whose range begins at or before pos; n_docs when there is none
__device__ __forceinline__ uint64_t doc_at(const uint64_t* __restrict__ offsets, uint64_t n_docs, uint64_t pos) {
    uint64_t lo = 0, hi = n_docs;  // offsets[lo - 1] <= pos < offsets[hi]
    while (lo < hi) {
        const uint64_t mid = (lo + hi) >> 1;
        if (offsets[mid] <= pos) lo = mid + 1;
        else hi = mid;
    }
    return lo ? lo - 1 : n_docs;
}

// the same for a whole wave and one position: 64 places are looked at together, three rounds where the above takes sixteen
__device__ __forceinline__ uint64_t wave_doc_at(const uint64_t* __restrict__ offsets, uint64_t n_docs, uint64_t pos) {
    const uint32_t lane = lane_id();
    uint64_t lo = 0, hi = n_docs;
    while (lo < hi) {
        const uint64_t step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step - 1;
        lo += step * (uint64_t)__popcll(__ballot(at < hi && offsets[at < hi ? at : lo] <= pos));
        if (step == 1) break;
        hi = hi < lo + step - 1 ? hi : lo + step - 1;
    }
    return lo ? lo - 1 : n_docs;
}

// documents of 64 positions in a row, lane by lane from p on: the first one's, and the begins behind it are searched in registers
__device__ __forceinline__ uint64_t wave_docs(const uint64_t* __restrict__ offsets, uint64_t n_docs, uint64_t p) {
    const uint32_t lane = lane_id();
    const uint64_t p0 = p - lane, d0 = wave_doc_at(offsets, n_docs, p0), next = d0 < n_docs ? d0 + 1 : 0;
    const uint64_t begin = next + lane < n_docs ? offsets[next + lane] - p0 : ~0ull;
    const uint32_t ahead = begin < 64 ? (uint32_t)begin : 64u;  // of p0, 64: behind all positions
    if (__shfl(ahead, 63, 64) < 64) return doc_at(offsets, n_docs, p);  // many documents are empty
    uint32_t c = 0;
#pragma unroll
    for (uint32_t step = 32; step; step >>= 1)
        if (__shfl(ahead, (int)(c + step - 1), 64) <= lane) c += step;
    return d0 < n_docs ? d0 + c : c ? c - 1 : n_docs;
}

template <typename O, int NS, bool NARROW>
__device__ __forceinline__ void store_cols(O* __restrict__ row, const uint32_t (&col)[NS], const bool (&in)[NS], uint32_t dim, const f32x8 (&v)[NS], float f) {
#pragma unroll
    for (int n = 0; n < NS; n++)
        if (in[n]) store8<O>(row + col[n], NARROW ? dim : 8, v[n] * f);
}

template <typename T, typename O, int NS, bool WEIGHTED, bool NARROW, bool ONCE>
__global__ __launch_bounds__(256) void pool_kernel(PoolArgs a) {
    const uint32_t lane = lane_id(), lpr = NS == 2 ? 64 : a.lpr;
    uint32_t block = blockIdx.x, blocks = gridDim.x, slab = blockIdx.y;
    if (NS == 1 && a.slabs > 1) {
        // one slab after the other down the list of blocks, an eighth of which each XCD takes in a row; and a slab's work in steps
        // of eight, so that each XCD has its part of the pieces, which come first and are the most work
        const uint32_t at = xcd_order(block, blocks);
        blocks /= a.slabs, slab = at / blocks, block = at - slab * blocks;
        const uint32_t run = blocks / 8;
        if (block < run * 8) block = block % run * 8 + block / run;
    }
    uint32_t col[NS];
    bool in[NS];
#pragma unroll
    for (int n = 0; n < NS; n++) {
        const uint32_t c = slab * (NS == 1 && a.slabs > 1 ? 256u : 512u * NS) + n * 512 + (lane & (lpr - 1)) * 8u;
        col[n] = lane_col<NARROW>(c, a.dim);
        in[n] = lane < lpr && c < a.dim;
    }
    const uint64_t n_work = a.n_pieces + a.n_docs, stride = (uint64_t)blocks * 4;
    const uint64_t piece = 1ull << a.piece_log2;
    for (uint64_t w = (uint64_t)block * 4 + threadIdx.x / 64; w < n_work; w += stride) {
        uint32_t n_named;
        f32x8 acc[NS];
        if (w < a.n_pieces) {  // shares of long documents
            const uint64_t lo = w << a.piece_log2, hi = lo + piece < a.n_ids ? lo + piece : a.n_ids;
            const uint64_t d0 = wave_doc_at(a.offsets, a.n_docs, lo), d1 = wave_doc_at(a.offsets, a.n_docs, hi - 1);
            uint64_t begins = ~0ull;
#pragma unroll 1
            for (int slot = 0; slot < 2; slot++) {
                const uint64_t d = slot ? d1 : d0;
                if (d >= a.n_docs || (slot && d1 == d0)) continue;
                uint64_t beg, end;
                doc_range(a.offsets, d, a.n_ids, beg, end);
                if (end - beg <= piece) continue;
                if (beg >= lo && beg < hi) begins = d;
                beg = beg > lo ? beg : lo;
                end = end < hi ? end : hi;
                sum_span<T, NS, WEIGHTED, NARROW, ONCE>(a, beg, end, col, acc, n_named);
                const uint64_t at = w * 2 + slot;
                store_cols<float, NS, NARROW>(a.part + at * a.dim, col, in, a.dim, acc, 1.0f);
                if (lane == 0 && slab == 0) a.part_n[at] = n_named;
            }
            if (lane == 0 && slab == 0) a.begins[w] = begins;
        } else {
            const uint64_t d = w - a.n_pieces;
            uint64_t beg, end;
            doc_range(a.offsets, d, a.n_ids, beg, end);
            if (a.n_pieces && end - beg > piece) continue;  // pool_join_kernel writes it
            sum_span<T, NS, WEIGHTED, NARROW, ONCE>(a, beg, end, col, acc, n_named);
            store_cols<O, NS, NARROW>(reinterpret_cast<O*>(a.out) + d * a.dim, col, in, a.dim, acc, pool_factor(a, n_named));
        }
    }
}

// A block per eight pieces and 512 columns. The long documents that begin in them are this block's: each of the four waves adds
// a quarter of its shares in order, eight at a time, and the quarters are added in order.
template <typename O, bool NARROW>
__global__ __launch_bounds__(256) void pool_join_kernel(PoolArgs a) {
    __shared__ __attribute__((aligned(32))) float quarter[3][512];
    const uint32_t lane = lane_id(), wave = threadIdx.x / 64, first_col = blockIdx.y * 512u + lane * 8u, col = lane_col<NARROW>(first_col, a.dim);
    const bool in = first_col < a.dim;
    const uint32_t wide = NARROW ? a.dim : 8;
    for (uint64_t base = (uint64_t)blockIdx.x * 8; base < a.n_pieces; base += (uint64_t)gridDim.x * 8) {
        const uint64_t mine = lane < 8 && base + lane < a.n_pieces ? a.begins[base + lane] : ~0ull;
        for (uint64_t left = __ballot(mine < a.n_docs); left; left &= left - 1) {  // the same for the whole block
            const int at = __ffsll((unsigned long long)left) - 1;
            const uint64_t first = base + at, d = __shfl(mine, at, 64);
            uint64_t beg, end;
            doc_range(a.offsets, d, a.n_ids, beg, end);
            const uint64_t last = (end - 1) >> a.piece_log2;
            // a long document leaves its first piece, so it is slot 0 there only if the piece begins with it
            const uint64_t at0 = first * 2 + (beg > first << a.piece_log2 ? 1 : 0);
            uint32_t n_named = 0;
            for (uint64_t k = first + lane; k <= last; k += 64) n_named += a.part_n[k == first ? at0 : k * 2];
#pragma unroll
            for (int m = 32; m; m >>= 1) n_named += __shfl_xor(n_named, m, 64);
            f32x8 acc = 0.0f;
            const float* __restrict__ part = a.part + col;
            const uint64_t each = (last - first + 4) / 4;  // shares first + [wave * each, (wave + 1) * each)
            uint64_t k = first + wave * each;
            const uint64_t stop = k + each < last + 1 ? k + each : last + 1;
            if (wave == 0) acc = load8<float>(part + at0 * a.dim, wide), k++;
            for (; k + 8 <= stop; k += 8) {
                f32x8 v[8];
#pragma unroll
                for (int u = 0; u < 8; u++) v[u] = load8<float>(part + (k + u) * 2 * a.dim, wide);
#pragma unroll
                for (int u = 0; u < 8; u++) acc += v[u];
            }
            for (; k < stop; k++) acc += load8<float>(part + k * 2 * a.dim, wide);
            if (wave) *reinterpret_cast<f32x8*>(&quarter[wave - 1][lane * 8]) = acc;
            __syncthreads();
            if (wave == 0 && in) {
#pragma unroll
                for (int q = 0; q < 3; q++) acc += *reinterpret_cast<const f32x8*>(&quarter[q][lane * 8]);
                store8<O>(reinterpret_cast<O*>(a.out) + d * a.dim + col, wide, acc * pool_factor(a, n_named));
            }
            __syncthreads();
        }
    }
}

// One row per id: eight rows per lane group in flight, read and written once -- bound by HBM: 262144 rows of 1024 in bf16 (131 MB
// of table, 537 MB of result) in 106 us, 6.3 TB/s, 161 with the result written through the caches; results that fit them stay
// there (262144 x 256 in 30 us).
template <typename T, bool NARROW, bool ONCE>
__global__ __launch_bounds__(256) void lookup_kernel(const T* __restrict__ table, uint64_t n_rows, uint32_t row_bytes, uint32_t dim, uint32_t lpr,
                                                     const void* __restrict__ ids, int id_bytes, uint64_t n_ids, float scale, T* __restrict__ out) {
    constexpr uint32_t U = 8;  // U * G positions per wave and round, 64 at most: lpr is 8 to 64
    const uint32_t G = 64 / lpr, lane = lane_id(), g = lane / lpr, c = blockIdx.y * 512u + (lane & (lpr - 1)) * 8u, col = lane_col<NARROW>(c, dim);
    const uint64_t stride = (uint64_t)gridDim.x * 4 * (U * G);
    for (uint64_t p = ((uint64_t)blockIdx.x * 4 + threadIdx.x / 64) * (U * G); p < n_ids; p += stride) {
        const uint32_t row = lane < U * G && p + lane < n_ids ? named_row(ids, id_bytes, p + lane, n_rows) : NO_ROW;
        uint32_t r[U];
        typename vec8<T>::raw raw[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) r[u] = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(u * G + g) * 4, (int)row);
#pragma unroll
        for (uint32_t u = 0; u < U; u++)
            raw[u] = load_cols<T, NARROW>(reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(table + col) + (uint64_t)(r[u] != NO_ROW ? r[u] : 0) * row_bytes), dim);
        if (c < dim) {
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
                if (p + u * G + g < n_ids) {
                    f32x8 v = __builtin_convertvector(raw[u], f32x8) * scale;
                    if (r[u] == NO_ROW) v = 0.0f;  // whatever row 0 and the scale hold
                    store8_or_once<T, ONCE>(out + (p + u * G + g) * dim + col, NARROW ? dim : 8, v);
                }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void fill_kernel(T* __restrict__ p, uint64_t n, T v) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) p[i] = v;
}

// ------------------------------------------------------------------------------------------ stable sort of (key, value)
// Least significant digit first, 8 bits a pass (262144 ids below 64000: two passes of 17 us). A wave ranks 64 keys at a time in
// their order: eight ballots give the lanes with the same digit, the ones below are the rank, a counter per wave and digit
// carries it on -- so equal keys keep their order and nothing depends on which wave runs first.
__device__ __forceinline__ uint32_t rank_digit(uint32_t digit, bool live, volatile uint32_t* counter) {  // volatile: other lanes write it
    uint64_t same = __ballot(live);
#pragma unroll
    for (int b = 0; b < 8; b++) {
        const uint64_t set = __ballot(live && (digit >> b & 1));
        same &= (digit >> b & 1) ? set : ~set;
    }
    uint32_t before = 0;
    if (live) before = counter[digit];
    const uint32_t rank = before + below(same);
    __builtin_amdgcn_wave_barrier();
    if (live && below(same) == 0) counter[digit] = before + (uint32_t)__popcll(same);
    __builtin_amdgcn_wave_barrier();
    return rank;
}

constexpr uint32_t SMALL_SORT = 8192;
// keys a block: 1024 up to 2^20 keys, so that a quarter of a million still fill the chip; 4096 beyond, for a shorter histogram
uint32_t sort_tile(uint64_t n) { return n <= (1u << 20) ? 1024 : 4096; }

__global__ __launch_bounds__(256) void sort_count_kernel(const uint32_t* __restrict__ key, uint32_t n, int shift, uint32_t tile, uint32_t n_tiles,
                                                         uint32_t* __restrict__ hist) {
    __shared__ uint32_t cnt[256];
    cnt[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * tile;
#pragma unroll 4
    for (uint32_t k = 0; k < tile; k += 256) {
        const uint32_t i = base + k + threadIdx.x;
        if (i < n) atomicAdd(&cnt[key[i] >> shift & 255u], 1u);
    }
    __syncthreads();
    hist[(uint64_t)threadIdx.x * n_tiles + blockIdx.x] = cnt[threadIdx.x];
}

// exclusive sum over the 256 threads of a block; *total = the sum
__device__ __forceinline__ uint32_t block_scan256(uint32_t v, uint32_t* lds4, uint32_t* total) {
    const uint32_t lane = lane_id(), wave = threadIdx.x / 64;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(s, d, 64);
        if (lane >= (uint32_t)d) s += o;
    }
    if (lane == 63) lds4[wave] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < 4; w++) {
        if (w < wave) before += lds4[w];
        all += lds4[w];
    }
    __syncthreads();
    *total = all;
    return before + s - v;
}

// block = digit: exclusive sums of its tile counts in place, their total behind the table
__global__ __launch_bounds__(256) void sort_scan_kernel(uint32_t* __restrict__ hist, uint32_t n_tiles) {
    __shared__ uint32_t lds4[4];
    uint32_t* row = hist + (uint64_t)blockIdx.x * n_tiles;
    uint32_t carry = 0;
    for (uint32_t k = 0; k < n_tiles; k += 256) {
        const uint32_t i = k + threadIdx.x, v = i < n_tiles ? row[i] : 0;
        uint32_t total;
        const uint32_t ex = block_scan256(v, lds4, &total);
        if (i < n_tiles) row[i] = carry + ex;
        carry += total;
    }
    if (threadIdx.x == 0) hist[(uint64_t)256 * n_tiles + blockIdx.x] = carry;
}

template <int PER>  // keys a thread
__global__ __launch_bounds__(256) void sort_scatter_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ val, uint32_t n, int shift,
                                                           uint32_t n_tiles, const uint32_t* __restrict__ hist, uint32_t* __restrict__ key_out,
                                                           uint32_t* __restrict__ val_out) {
    __shared__ uint32_t cnt[4][256], lds4[4];
    const uint32_t t = threadIdx.x, wave = t / 64, lane = lane_id();
    for (int w = 0; w < 4; w++) cnt[w][t] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * (PER * 256) + wave * (PER * 64) + lane;
    uint32_t k_[PER], rank[PER];
#pragma unroll
    for (int r = 0; r < PER; r++) k_[r] = base + r * 64 < n ? key[base + r * 64] : 0;
#pragma unroll
    for (int r = 0; r < PER; r++) rank[r] = rank_digit(k_[r] >> shift & 255u, base + r * 64 < n, cnt[wave]);
    __syncthreads();
    uint32_t all;
    uint32_t at = block_scan256(hist[(uint64_t)256 * n_tiles + t], lds4, &all) + hist[(uint64_t)t * n_tiles + blockIdx.x];
    for (int w = 0; w < 4; w++) {
        const uint32_t c = cnt[w][t];
        cnt[w][t] = at;
        at += c;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < PER; r++)
        if (base + r * 64 < n) {
            const uint32_t to = cnt[wave][k_[r] >> shift & 255u] + rank[r];
            if (to < n) {  // always, unless the keys change while they are sorted
                key_out[to] = k_[r];
                val_out[to] = val[base + r * 64];
            }
        }
}

// What the gradient sorts.  key = id, or n_rows for padding and for positions outside every document; val = the row of the
// gradient that the position's table row took part in.  With count given, the documents' named ids are counted (whole
// numbers: the order of the atomics does not matter; one atomic per document that a wave's positions lie in).
struct GradIds {
    const void* ids;
    int id_bytes;
    uint64_t n_ids, n_rows;
    const uint64_t* offsets;
    uint64_t n_docs;
    uint32_t* count;
};
__device__ __forceinline__ void grad_key(const GradIds& g, uint64_t p, uint32_t& key, uint32_t& val) {  // call with all lanes
    uint64_t row = p;
    uint32_t id = NO_ROW;
    bool named = false;
    const uint64_t doc = g.offsets ? wave_docs(g.offsets, g.n_docs, p) : 0;
    if (p < g.n_ids) {
        id = named_row(g.ids, g.id_bytes, p, g.n_rows);
        named = id != NO_ROW;
        if (g.offsets) {
            row = doc;
            uint64_t beg = 0, end = 0;
            if (row < g.n_docs) doc_range(g.offsets, row, g.n_ids, beg, end);
            if (p < beg || p >= end) named = false;
        }
    }
    key = named ? id : (uint32_t)g.n_rows;
    val = named ? (uint32_t)row : 0u;
    if (!g.count) return;
    const uint64_t live = __ballot(named);
    if (!live) return;
    for (uint64_t left = live; left;) {
        const int leader = __ffsll((unsigned long long)left) - 1;
        const uint32_t first = __shfl((uint32_t)row, leader, 64);
        const uint64_t same = __ballot(named && (uint32_t)row == first);
        if ((int)lane_id() == leader) atomicAdd(&g.count[first], (uint32_t)__popcll(same));
        left &= ~same;
    }
}

// Up to SMALL_SORT pairs in one block and one launch, all passes in LDS: 450 edges 10 us, 6750 30 (four passes each). Counting
// for each edge on all CUs how many are before it takes 16 for 6750, but a workspace and a launch more, which cost the few edges of
// a small search 3 us; a choice by the number of edges is not made yet. val_bits > 0: by the value's bits first, then by the
// key's. MAKE: the pairs are the gradient's, made on the way in
template <bool MAKE>
__global__ __launch_bounds__(1024) void small_sort_kernel(uint32_t* __restrict__ key, uint32_t* __restrict__ val, uint32_t n, int val_bits, int bits, GradIds g) {
    __shared__ uint32_t ks[SMALL_SORT], vs[SMALL_SORT], cnt[16][256], lds4[4];
    const uint32_t t = threadIdx.x, wave = t / 64, lane = lane_id();
    const uint32_t rounds = (n + 1023) / 1024, base = wave * rounds * 64 + lane;  // of 64 pairs a wave, all sixteen waves at work
    uint32_t k_[8], v_[8], rank[8];
#pragma unroll
    for (int r = 0; r < 8; r++) {
        const uint32_t i = base + r * 64;
        k_[r] = v_[r] = 0;
        if (r < (int)rounds) {
            if (MAKE) grad_key(g, i, k_[r], v_[r]);
            else if (i < n) k_[r] = key[i], v_[r] = val[i];
        }
    }
    for (int pass = 0, passes = (val_bits + 7) / 8 + (bits + 7) / 8; pass < passes; pass++) {
        const bool by_val = pass < (val_bits + 7) / 8;
        const int shift = 8 * (by_val ? pass : pass - (val_bits + 7) / 8);
        for (uint32_t i = t; i < 16 * 256; i += 1024) (&cnt[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 8; r++)
            if (r < (int)rounds) rank[r] = rank_digit((by_val ? v_[r] : k_[r]) >> shift & 255u, base + r * 64 < n, cnt[wave]);
        __syncthreads();
        uint32_t own = 0;
        if (t < 256)
            for (int w = 0; w < 16; w++) own += cnt[w][t];
        uint32_t ex = own;
        if (wave < 4) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t o = __shfl_up(ex, d, 64);
                if (lane >= (uint32_t)d) ex += o;
            }
            if (lane == 63) lds4[wave] = ex;
        }
        __syncthreads();
        if (t < 256) {
            uint32_t at = ex - own;
            for (uint32_t w = 0; w < wave; w++) at += lds4[w];
            for (int w = 0; w < 16; w++) {
                const uint32_t c = cnt[w][t];
                cnt[w][t] = at;
                at += c;
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 8; r++)
            if (r < (int)rounds && base + r * 64 < n) {
                const uint32_t to = cnt[wave][(by_val ? v_[r] : k_[r]) >> shift & 255u] + rank[r];
                ks[to] = k_[r];
                vs[to] = v_[r];
            }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const uint32_t i = base + r * 64;
            if (r < (int)rounds && i < n) k_[r] = ks[i], v_[r] = vs[i];
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < 8; r++)
        if (r < (int)rounds && base + r * 64 < n) {
            key[base + r * 64] = k_[r];
            val[base + r * 64] = v_[r];
        }
}

int bits_of(uint64_t largest) {
    int b = 1;
    while (b < 64 && largest >> b) b++;
    return b;
}
uint64_t sort_hist_words(uint64_t n) { return n <= SMALL_SORT ? 0 : 256 * ((n + sort_tile(n) - 1) / sort_tile(n)) + 256; }
// More than SMALL_SORT pairs: sorts (key, val) by key, the values of equal keys in their order.  (key2, val2) are scratch of the
// same length; the result is in key / val, which change places with key2 / val2 in every pass
void sort_pairs(hipStream_t s, uint32_t*& key, uint32_t*& val, uint32_t*& key2, uint32_t*& val2, uint64_t n, int bits, uint32_t* hist) {
    const uint32_t tile = sort_tile(n), tiles = (uint32_t)((n + tile - 1) / tile);
    auto scatter = tile == 1024 ? sort_scatter_kernel<4> : sort_scatter_kernel<16>;
    for (int shift = 0; shift < bits; shift += 8) {
        hipLaunchKernelGGL(sort_count_kernel, dim3(tiles), dim3(256), 0, s, key, (uint32_t)n, shift, tile, tiles, hist);
        hipLaunchKernelGGL(sort_scan_kernel, dim3(256), dim3(256), 0, s, hist, tiles);
        hipLaunchKernelGGL(scatter, dim3(tiles), dim3(256), 0, s, key, val, (uint32_t)n, shift, tiles, hist, key2, val2);
        std::swap(key, key2);
        std::swap(val, val2);
    }
}

// ------------------------------------------------------------------------------------------------ gradient of the lookup
// one thread a position, for more than small_sort_kernel takes
__global__ __launch_bounds__(256) void grad_keys_kernel(GradIds g, uint32_t* __restrict__ key, uint32_t* __restrict__ val) {
    const uint64_t p = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    uint32_t k, v;
    grad_key(g, p, k, v);
    if (p < g.n_ids) key[p] = k, val[p] = v;
}

// start[v] = first sorted position with a key >= v, v = 0 .. n_rows
__global__ __launch_bounds__(256) void grad_starts_kernel(const uint32_t* __restrict__ key, uint32_t n, uint64_t n_rows, uint64_t* __restrict__ start) {
    const uint64_t v = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (v > n_rows) return;
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (key[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    start[v] = lo;
}

// ------------------------------------------------------------------------------------------------ launching the sums
uint32_t piece_log2_for(uint64_t n_ids) {
    // A document of all ids takes a wave's time for a piece, then a quarter of its n_ids / piece shares: shortest with pieces of
    // sqrt(n_ids) / 2.  32 to 1024 ids: fewer would make the shares as many as the rows, more gains nothing
    uint32_t b = 5;
    while (b < 10 && (4ull << (2 * b)) < n_ids) b++;
    return b;
}
uint64_t n_pieces_for(uint64_t n_ids) {
    const uint32_t b = piece_log2_for(n_ids);
    return n_ids <= (1ull << b) ? 0 : (n_ids + (1ull << b) - 1) >> b;  // none is long where all ids fit one piece
}
uint64_t pool_ws_bytes(uint64_t n_ids, uint32_t dim) {
    const uint64_t p = n_pieces_for(n_ids);
    return p ? round_up(p * 2 * dim * 4, 256) + round_up(p * 2 * 4, 256) + round_up(p * 8, 256) : 0;
}
void place_parts(PoolArgs& a, uint8_t* ws) {
    a.part = reinterpret_cast<float*>(ws);
    a.part_n = reinterpret_cast<uint32_t*>(ws + round_up(a.n_pieces * 2 * a.dim * 4, 256));
    a.begins = reinterpret_cast<uint64_t*>(ws + round_up(a.n_pieces * 2 * a.dim * 4, 256) + round_up(a.n_pieces * 2 * 4, 256));
}

uint32_t lanes_per_row(uint32_t dim) { return dim > 256 ? 64 : dim > 128 ? 32 : dim > 64 ? 16 : 8; }

// Every XCD has an L2 of 4 MB of its own.  With a row's columns shared out among them, 256 a slab, an L2 keeps its slab of the
// table instead of a little of everything: 10000 documents of 480 ids, 64000 x 1024 in bf16, 630 -> 488 us; 30000 of 64 ids,
// 64000 x 768 in fp32, 441 -> 338. Not where a slab would be mostly empty, where the table fits or its rows are not named
// again, or where sums are so short that reading their ids once a slab costs more (10 ids a document: 315 us whole, 487 in
// slabs; at 32 ids 259 and 253). Slabs of 128 columns: 40000 documents of 480 x 256 531 us instead of 497.
uint32_t column_slabs(const PoolArgs& a) {
    const uint32_t n = (a.dim + 255) / 256;
    if (n < 2 || n * 256 > a.dim + a.dim / 8 || a.n_rows * a.row_bytes <= (4u << 20) || a.n_ids < 2 * a.n_rows || a.n_ids < 32 * a.n_docs) return 1;
    return n;
}

template <typename T, typename O, bool WEIGHTED, bool ONCE>
void launch_pool(hipStream_t s, PoolArgs a) {
    a.slabs = column_slabs(a);
    if (a.slabs > 1) a.lpr = 32;
    const uint32_t ns = a.dim > 512 && a.slabs == 1 ? 2 : 1, slabs = a.slabs > 1 ? a.slabs : (a.dim + 512 * ns - 1) / (512 * ns);
    const uint64_t cap = (1u << 20) / slabs + 1, want = (a.n_pieces + a.n_docs + 3) / 4, blocks = want < cap ? want : cap;
    const dim3 grid((unsigned)(a.slabs > 1 ? blocks * slabs : blocks), a.slabs > 1 ? 1 : slabs), block(256);
    if (a.dim < 8) hipLaunchKernelGGL((pool_kernel<T, O, 1, WEIGHTED, true, false>), grid, block, 0, s, a);
    else if (ns == 2) hipLaunchKernelGGL((pool_kernel<T, O, 2, WEIGHTED, false, ONCE>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((pool_kernel<T, O, 1, WEIGHTED, false, ONCE>), grid, block, 0, s, a);
    if (a.n_pieces) {
        const uint32_t slabs = (a.dim + 511) / 512;
        const uint64_t cap = (1u << 20) / slabs + 1;
        auto join = a.dim < 8 ? pool_join_kernel<O, true> : pool_join_kernel<O, false>;
        hipLaunchKernelGGL(join, dim3((unsigned)((a.n_pieces + 7) / 8 < cap ? (a.n_pieces + 7) / 8 : cap), slabs), dim3(256), 0, s, a);
    }
}

template <typename T>
void launch_lookup(hipStream_t s, const T* table, uint64_t n_rows, uint64_t stride, uint32_t dim, const void* ids, int id_bytes, uint64_t n_ids, float scale, T* out) {
    const uint32_t slabs = (dim + 511) / 512, lpr = lanes_per_row(dim);
    const uint64_t per_block = 4ull * (64 / lpr) * 8, cap = (1u << 22) / slabs + 1, want = (n_ids + per_block - 1) / per_block;
    const dim3 grid((unsigned)(want < cap ? want : cap), slabs), block(256);
    auto kernel = dim < 8 ? lookup_kernel<T, true, false> : n_ids * dim * sizeof(T) <= LAST_LEVEL ? lookup_kernel<T, false, false> : lookup_kernel<T, false, true>;
    hipLaunchKernelGGL(kernel, grid, block, 0, s, table, n_rows, (uint32_t)(stride * sizeof(T)), dim, lpr, ids, id_bytes, n_ids, scale, out);
}

// ------------------------------------------------------------------------------------------------ norm
// A row is held in registers, 8 * NC columns a lane, by L lanes: 16 to 64 up to 2048 columns (no barrier; 256 / L rows a block), four
// waves up to 8192, sixteen beyond.  x is read once and everything written once: bound by HBM.  20001 x 1000 in fp16 with
// residual 29 us (5.5 TB/s, part of it from the last-level cache); 262144 x 768 in bf16 with residual 265 us past the caches, 290
// through them, 8000 x 4096 39 us through and 46 past.  Into 8 bits 262144 x 768 with residual 266 us, 5.3 TB/s, without 172, into
// e4m3 241: there the arithmetic in 64 bits bounds it.
//
// As in the lookup, a lane's eight columns never reach over the row's end: the last lane starts early enough and overlaps its
// neighbour, and lanes behind it read the same eight and store nothing.  So no load stands behind a branch and all of a row's are
// on their way at once (with a branch for the end, one after the other: 262144 x 770 in bf16 185 us, so 137).
// What a lane repeats is left out of the sums.  Rows narrower than eight (NARROW) take single elements.
template <bool NARROW>
struct Eight {
    uint32_t at, skip;  // first column; how many of the eight belong to lanes before
    bool in;            // whether any is this lane's own
    __device__ __forceinline__ Eight(uint32_t lane_of_row, uint32_t dim) {
        const uint32_t col = lane_of_row * 8;
        in = col < dim;
        at = NARROW ? 0 : col < dim - 8 ? col : dim - 8;
        skip = NARROW ? 0 : col - at;
    }
    template <typename T, bool ONCE>
    __device__ __forceinline__ f32x8 load(const T* __restrict__ row, uint32_t dim) const {
        const auto* p = reinterpret_cast<const typename vec8<T>::raw_any*>(row + at);
        if constexpr (NARROW) return load8<T>(row, dim);
        else if constexpr (ONCE) return __builtin_convertvector(__builtin_nontemporal_load(p), f32x8);
        else return __builtin_convertvector(*p, f32x8);
    }
    template <typename T, bool ONCE>
    __device__ __forceinline__ void store(T* __restrict__ row, uint32_t dim, f32x8 v) const {
        if (in) store8_or_once<T, ONCE>(row + at, NARROW ? dim : 8, v);
    }
    // sum of a[k] * b[k] over this lane's own
    __device__ __forceinline__ float dot(f32x8 a, f32x8 b, uint32_t dim) const {
        float s = 0;
        if (!NARROW && dim % 8) {
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) s = fmaf(k >= skip ? a[k] : 0.0f, k >= skip ? b[k] : 0.0f, s);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) s = fmaf(a[k], b[k], s);
        }
        return in ? s : 0.0f;
    }
};
constexpr int waves_of(int l) { return l <= 64 ? 1 : l / 64; }
template <int L>
__device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
    for (int m = (L < 64 ? L : 64) / 2; m; m >>= 1) v += __shfl_xor(v, m, 64);
    if (L <= 64) return v;
    if (lane_id() == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    float s = 0;
#pragma unroll
    for (int w = 0; w < waves_of(L); w++) s += lds[w];
    __syncthreads();
    return s;
}
template <int L, typename F>
__device__ __forceinline__ F row_max(F v, F* lds) {
#pragma unroll
    for (int m = (L < 64 ? L : 64) / 2; m; m >>= 1) {
        const F o = __shfl_xor(v, m, 64);
        v = v > o ? v : o;
    }
    if (L <= 64) return v;
    if (lane_id() == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < waves_of(L); w++) v = v > lds[w] ? v : lds[w];
    __syncthreads();
    return v;
}

// 1 / sqrt(m): the hardware's reciprocal root, a unit of the last place off, and one step of Newton's iteration in 64 bits
__device__ __forceinline__ double inverse_root(float m) {
    if (!(m >= 0x1p-126f && m <= 0x1p126f)) return 1.0f / sqrtf(m);  // zeros and infinities among them
    const double x = __builtin_amdgcn_rsqf(m);
    return fma(0.5 * x, fma(-(double)m * x, x, 1.0), x);
}

// A row whose squares do not add up to a 32-bit number: they are lost (below 2^-126, which counts where eps does not cover them)
// or overflow.  Such a row is read and summed again, with the larger of its largest element and eps's root scaled to [0.5, 1).  It
// is a rare one and goes element by element, from a lane number that the compiler cannot see through, so that nothing of this
// is worked out ahead for all rows: they pay 4 % at most (20001 x 1000 fp16 to int8 19.2 -> 20.0 us, 262144 x 768 none).  Sums of
// squares in 64 bits, which need no second reading, cost 10 to 40 % (8000 x 4096 fp32 to int8 30 -> 33 us, 4000 x 8192 bf16 32 -> 44).
__device__ __forceinline__ bool off_range(float squares, float m) { return !(m >= 0x1p-100f && squares < __builtin_inff()); }
__device__ __forceinline__ uint32_t unseen(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}
template <typename T>
__device__ __forceinline__ float sum_at(const T* __restrict__ x, const T* __restrict__ res, uint32_t c) {
    return (float)x[c] + (res ? (float)res[c] : 0.0f);
}
// mean = (mean of the squares + eps) * 2^-2e.  false for rows of zeros, with an infinity, or of NaN only: they stay as they are.
// Call with all lanes of the row, of which this is lane t
template <typename T, int L>
__device__ __forceinline__ bool row_again(const T* __restrict__ x, const T* __restrict__ res, uint32_t t, uint32_t dim, float eps, float* lds, float& mean, int& e) {
    float big = 0, ss = 0;
#pragma unroll 1
    for (uint32_t c = t; c < dim; c += L) big = fmaxf(big, fabsf(sum_at<T>(x, res, c)));
    big = row_max<L>(big, lds);
    if (!(big > 0.0f && big < __builtin_inff())) return false;
    e = __builtin_amdgcn_frexp_expf(fmaxf(big, __builtin_amdgcn_sqrtf(eps)));
#pragma unroll 1
    for (uint32_t c = t; c < dim; c += L) {
        const float h = ldexpf(sum_at<T>(x, res, c), -e);
        ss = fmaf(h, h, ss);
    }
    mean = row_sum<L>(ss, lds) / (float)dim + ldexpf(eps, -2 * e);
    return true;
}

template <typename T, int NC, int L, bool NARROW, bool ONCE>
__global__ __launch_bounds__(L == 1024 ? 1024 : 256) void norm_kernel(const T* __restrict__ x, uint64_t xs, const T* __restrict__ res, uint64_t rs,
                                                                    const T* __restrict__ weight, float eps, uint64_t n, uint32_t dim, T* __restrict__ y,
                                                                    T* __restrict__ sum_out, float* __restrict__ rstd) {
    constexpr uint32_t RPB = L <= 64 ? 256 / L : 1;  // rows a block
    __shared__ float lds[waves_of(L)];
    const uint32_t t = threadIdx.x % L;
    for (uint64_t row = (uint64_t)blockIdx.x * RPB + threadIdx.x / L; row < n; row += (uint64_t)gridDim.x * RPB) {
        f32x8 h[NC], w[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) h[c] = Eight<NARROW>(c * L + t, dim).template load<T, ONCE>(x + row * xs, dim), w[c] = 1.0f;
        if (weight) {
#pragma unroll
            for (int c = 0; c < NC; c++) w[c] = Eight<NARROW>(c * L + t, dim).template load<T, false>(weight, dim);
        }
        if (res) {
#pragma unroll
            for (int c = 0; c < NC; c++) h[c] += Eight<NARROW>(c * L + t, dim).template load<T, ONCE>(res + row * rs, dim);
        }
        float ss = 0;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const Eight<NARROW> own(c * L + t, dim);
            if (sum_out) own.template store<T, ONCE>(sum_out + row * dim, dim, h[c]);
            ss += own.dot(h[c], h[c], dim);
        }
        const float squares = row_sum<L>(ss, lds), m = squares / (float)dim + eps;
        if (off_range(squares, m)) {  // the same for the whole row
            const uint32_t lane = unseen(t);
            const T *xr = x + row * xs, *rr = res ? res + row * rs : nullptr;
            int e;
            float mean;
            if (row_again<T, L>(xr, rr, lane, dim, eps, lds, mean, e)) {
                const float root = (float)inverse_root(mean);
                if (rstd && lane == 0) rstd[row] = ldexpf(root, -e);
#pragma unroll 1
                for (uint32_t c = lane; c < dim; c += L) y[row * dim + c] = (T)(ldexpf(sum_at<T>(xr, rr, c), -e) * root * (weight ? (float)weight[c] : 1.0f));
                continue;
            }
        }
        const float r = (float)inverse_root(m);
        if (rstd && t == 0) rstd[row] = r;
#pragma unroll
        for (int c = 0; c < NC; c++) Eight<NARROW>(c * L + t, dim).template store<T, ONCE>(y + row * dim, dim, h[c] * r * w[c]);
    }
}

// The nearest 8-bit value to z = y * top / big.  zf is z rounded to 32 bits, at most 2^-24 of its size off, which is below
// 1e-5 of a step; only next to a midpoint (near_tie) does exact arithmetic decide: whether y * top is above the midpoint times
// big, the two products' difference taken without a rounding that could change its sign.  So the codes do not depend on how the
// row was summed, without a division per element.
template <int KIND>
__device__ __forceinline__ float step8(float zf) {  // from one 8-bit value to the next, as 1 / step: a power of two
    if (KIND == MDD_I8) return 1.0f;
    const uint32_t e = __float_as_uint(zf) >> 23 & 255u;
    return __uint_as_float((254u + 3u - (e > 121u ? e : 121u)) << 23);  // three bits behind the leading one, 2^-9 below 2^-6
}
template <int KIND>
__device__ __forceinline__ bool near_tie(float zf) {
    const float u = zf * step8<KIND>(zf), whole = 12582912.0f;  // 1.5 * 2^23: a sum with it is rounded to a whole number
    return fabsf(u - ((u + whole) - whole)) >= 0.49998f;
}
template <int KIND>
__device__ __forceinline__ float nearest8_exact(float zf, double y, double big) {
    const float inv = step8<KIND>(zf), f = floorf(zf * inv);
    const double top = KIND == MDD_I8 ? 127.0 : 448.0, mid = ((double)f + 0.5) / (double)inv;
    const double p = mid * big, d = fma(y, top, -p) - fma(mid, big, -p);
    const bool up = d > 0.0 || (d == 0.0 && floorf(f * 0.5f) * 2.0f != f);  // between two, to the even one
    return (up ? f + 1.0f : f) / inv;
}

// (Three waves a SIMD with four pieces of a row a lane: left alone the compiler takes 171 registers instead of 168, 35 -> 41 us at 20000 x
// 2048 in fp32.)
template <typename T, int NC, int L, int KIND, bool NARROW, bool ONCE>
__global__ __launch_bounds__(L == 1024 ? 1024 : 256, L == 1024 ? 4 : NC == 4 ? 3 : 1) void norm_q8_kernel(const T* __restrict__ x, uint64_t xs, const T* __restrict__ res, uint64_t rs,
                                                                       const T* __restrict__ weight, float eps, uint64_t n, uint32_t dim,
                                                                       uint8_t* __restrict__ codes, float* __restrict__ scales, T* __restrict__ sum_out) {
    constexpr uint32_t RPB = L <= 64 ? 256 / L : 1;  // rows a block
    __shared__ float lds[waves_of(L)];
    __shared__ double ldsd[waves_of(L)];
    const uint32_t t = threadIdx.x % L;
    const double top = KIND == MDD_I8 ? 127.0 : 448.0;
    for (uint64_t row = (uint64_t)blockIdx.x * RPB + threadIdx.x / L; row < n; row += (uint64_t)gridDim.x * RPB) {
        double y[NC][8];  // h * weight: a sum and a product of 8 to 24-bit numbers, exact in 64 bits unless the two of the sum lie far apart
        f32x8 v[NC], o[NC], w[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) v[c] = Eight<NARROW>(c * L + t, dim).template load<T, ONCE>(x + row * xs, dim), o[c] = 0.0f, w[c] = 1.0f;
        if (res) {
#pragma unroll
            for (int c = 0; c < NC; c++) o[c] = Eight<NARROW>(c * L + t, dim).template load<T, ONCE>(res + row * rs, dim);
        }
        if (weight) {
#pragma unroll
            for (int c = 0; c < NC; c++) w[c] = Eight<NARROW>(c * L + t, dim).template load<T, false>(weight, dim);
        }
        float ss = 0;
        double big = 0;
        bool bad = false;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const Eight<NARROW> own(c * L + t, dim);
            const f32x8 h = v[c] + o[c];
            if (sum_out) own.template store<T, ONCE>(sum_out + row * dim, dim, h);
            ss += own.dot(h, h, dim);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                y[c][k] = ((double)v[c][k] + (double)o[c][k]) * (double)w[c][k];
                bad |= !(fabs(y[c][k]) < __builtin_inf());
                big = fmax(big, fabs(y[c][k]));
            }
        }
        if (bad) big = __builtin_inf();  // fmax drops a NaN: an infinity stands for both
        big = row_max<L>(big, ldsd);
        const float squares = row_sum<L>(ss, lds), m = squares / (float)dim + eps;
        const bool fine = big < __builtin_inf(), off = off_range(squares, m);
        if (t == 0) scales[row] = !fine ? __builtin_nanf("") : big > 0 ? (float)(big * (inverse_root(m) * (1.0 / top))) : 0.0f;
        const double inv = big > 0 ? top / big : 0.0;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const Eight<NARROW> own(c * L + t, dim);
            if (!own.in) continue;
            uint32_t pack[2] = {0, 0};
            if (fine && big > 0) {
                float z[8];
                bool tie[8], any = false;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    z[k] = (float)(y[c][k] * inv);
                    tie[k] = near_tie<KIND>(z[k]);
                    any |= tie[k];
                }
                if (any) {
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (tie[k]) z[k] = nearest8_exact<KIND>(z[k], y[c][k], big);
                }
#pragma unroll
                for (int k = 0; k < 8; k += 4) {
                    if (KIND == MDD_I8) {
                        uint32_t b[4];  // the low byte of the sum is the whole number's
#pragma unroll
                        for (int l = 0; l < 4; l++) b[l] = __float_as_uint(z[k + l] + 12582912.0f);
                        const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u);
                        pack[k / 4] = hi << 16 | lo;
                    } else {
                        const int p = __builtin_amdgcn_cvt_pk_fp8_f32(z[k], z[k + 1], 0, false);  // to the nearest
                        pack[k / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[k + 2], z[k + 3], p, true);
                    }
                }
            }
            uint8_t* to = codes + row * dim + own.at;
            if constexpr (!NARROW) {
                typedef uint32_t pair_any __attribute__((ext_vector_type(2), aligned(1)));
                const pair_any v = {pack[0], pack[1]};
                if (ONCE) __builtin_nontemporal_store(v, reinterpret_cast<pair_any*>(to));
                else *reinterpret_cast<pair_any*>(to) = v;
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 8; k++)
                    if (k < dim) to[k] = (uint8_t)(pack[k / 4] >> (8 * (k % 4)));
            }
        }
        if (off && fine && big > 0) {  // the same for the whole row: its scale once more
            const uint32_t lane = unseen(t);
            int e;
            float mean;
            if (row_again<T, L>(x + row * xs, res ? res + row * rs : nullptr, lane, dim, eps, lds, mean, e) && lane == 0)
                scales[row] = (float)(big * (ldexp(inverse_root(mean), -e) * (1.0 / top)));
        }
    }
}

// Backward: a fixed number of blocks walks the rows; the weight's gradient stays in registers over a block's rows, goes to a
// workspace row per block and is added up by weight_grad_kernel in block order.  20001 x 1000 in fp16: 30 us with four blocks a CU
// (43 with two: too few loads in flight), and 5 for the join.
template <typename T, int NC, int L, bool NARROW>
__global__ __launch_bounds__(L == 1024 ? 1024 : 256) void norm_backward_kernel(const T* __restrict__ g, uint64_t gs, const T* __restrict__ h, uint64_t hs,
                                                                             const T* __restrict__ gsum, uint64_t gss, const T* __restrict__ weight,
                                                                             const float* __restrict__ rstd, uint64_t n, uint32_t dim, T* __restrict__ dx,
                                                                             float* __restrict__ part) {
    constexpr uint32_t RPB = L <= 64 ? 256 / L : 1;  // rows a block
    __shared__ float lds[waves_of(L)];
    __shared__ __attribute__((aligned(32))) float across[RPB > 1 ? (RPB - 1) * L * 8 : 8];
    const uint32_t t = threadIdx.x % L, sub = threadIdx.x / L;
    f32x8 w[NC], dw[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        w[c] = 1.0f, dw[c] = 0.0f;
        if (weight) w[c] = Eight<NARROW>(c * L + t, dim).template load<T, false>(weight, dim);
    }
    for (uint64_t row = (uint64_t)blockIdx.x * RPB + sub; row < n; row += (uint64_t)gridDim.x * RPB) {
        const float r = rstd[row];
        f32x8 nx[NC], gw[NC], more[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const Eight<NARROW> own(c * L + t, dim);
            nx[c] = own.template load<T, false>(h + row * hs, dim);
            gw[c] = own.template load<T, false>(g + row * gs, dim);
        }
        if (gsum) {
#pragma unroll
            for (int c = 0; c < NC; c++) more[c] = Eight<NARROW>(c * L + t, dim).template load<T, false>(gsum + row * gss, dim);
        }
        float dot = 0;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            nx[c] *= r;
            dw[c] += gw[c] * nx[c];
            gw[c] *= w[c];
            dot += Eight<NARROW>(c * L + t, dim).dot(gw[c], nx[c], dim);
        }
        const float mean = row_sum<L>(dot, lds) / (float)dim;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            f32x8 v = (gw[c] - nx[c] * mean) * r;
            if (gsum) v += more[c];
            Eight<NARROW>(c * L + t, dim).template store<T, false>(dx + row * dim, dim, v);
        }
    }
    if (!part) return;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        if (RPB > 1) {
            if (sub) *reinterpret_cast<f32x8*>(&across[((sub - 1) * L + t) * 8]) = dw[c];
            __syncthreads();
            if (!sub)
                for (uint32_t s = 0; s < RPB - 1; s++) dw[c] += *reinterpret_cast<const f32x8*>(&across[(s * L + t) * 8]);
            __syncthreads();
        }
        if (sub == 0) Eight<NARROW>(c * L + t, dim).template store<float, false>(part + (uint64_t)blockIdx.x * dim, dim, dw[c]);
    }
}

// 64 columns a block, its 16 waves take every 16th workspace row
__global__ __launch_bounds__(1024) void weight_grad_kernel(const float* __restrict__ part, uint32_t n_parts, uint32_t dim, float* __restrict__ out) {
    __shared__ float lds[16][64];
    const uint32_t lane = lane_id(), wave = threadIdx.x / 64, col = blockIdx.x * 64 + lane;
    float s = 0;
    if (col < dim) {
#pragma unroll 8
        for (uint32_t p = wave; p < n_parts; p += 16) s += part[(uint64_t)p * dim + col];
    }
    lds[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < dim) {
        s = 0;
#pragma unroll
        for (int w = 0; w < 16; w++) s += lds[w][lane];
        out[col] = s;
    }
}

// Picks NC, L and NARROW of a row kernel, 8 * NC * L columns: body(NC, L, NARROW) as integral constants.  Up to 2048 columns the lanes
// that hold a row with the fewest idle: 262144 x 768 in bf16 to int8 by 32 lanes with 24 columns each 200 us, by 64 with 16 258;
// 100000 x 100 by 16 lanes 16 us, by 64 52.  Beyond, for 4096 columns, 8192 and so on: up to half of the lanes are idle there, of which a
// plain norm feels 6 % (24000 x 5120 in bf16 6.0 TB/s, x 8192 6.4).
template <typename F>
auto for_width(uint32_t dim, bool backward, F&& body) {
    auto pick = [&](auto nc, auto l) { return body(nc, l, std::false_type()); };
    typedef std::integral_constant<int, 1> one;
    typedef std::integral_constant<int, 2> two;
    typedef std::integral_constant<int, 3> three;
    typedef std::integral_constant<int, 4> four;
    if (dim < 8) return body(one(), std::integral_constant<int, 16>(), std::true_type());
    if (dim <= 128) return pick(one(), std::integral_constant<int, 16>());
    if (dim <= 256) return pick(one(), std::integral_constant<int, 32>());
    if (dim <= 384 && !backward) return pick(three(), std::integral_constant<int, 16>());  // (50000 x 384 28 -> 21 us; backward 25 -> 29)
    if (dim <= 512) return pick(one(), std::integral_constant<int, 64>());
    if (dim <= 768) return pick(three(), std::integral_constant<int, 32>());
    if (dim <= 1024) return pick(two(), std::integral_constant<int, 64>());
    if (dim <= 1536) return pick(three(), std::integral_constant<int, 64>());
    if (dim <= 2048) return pick(four(), std::integral_constant<int, 64>());
    if (dim <= 4096) return pick(two(), std::integral_constant<int, 256>());
    if (dim <= 8192) return pick(four(), std::integral_constant<int, 256>());
    if (dim <= 16384) return pick(two(), std::integral_constant<int, 1024>());
    return pick(four(), std::integral_constant<int, 1024>());
}
uint64_t row_blocks(uint64_t n, int l) { return l <= 64 ? (n * l + 255) / 256 : n; }
dim3 row_grid(uint64_t n, int l) {
    const uint64_t want = row_blocks(n, l);
    return dim3((unsigned)(want < (1u << 20) ? want : (1u << 20)));
}
uint32_t backward_blocks(uint64_t n, uint32_t dim) {
    const uint64_t want = for_width(dim, true, [&](auto, auto l, auto) { return row_blocks(n, l.value); });
    return (uint32_t)(want < 1024 ? want : 1024);  // four blocks a CU
}

// ------------------------------------------------------------------------------------------------ edge cosines
// L lanes take an edge, 16 columns each and four times that in flight, of both rows: 16 lanes, or fewer for rows below 128 bytes.
// Bound by the gather of two rows per edge: 2 million random edges on 262144 x 768 bytes (201 MB, the last-level cache) in
// 410 us, 7.5 TB/s, the rate at which lines that miss L2 arrive; with one chunk in flight instead of four it is the same.
// As elsewhere here the last lane's 16 bytes overlap its neighbour's, so that no load stands behind a branch, and what it
// repeats is masked out (1 million edges of 250 bytes 111 us, with a branch for the end and always 16 lanes
// 320; of 128 bytes 40 and 84).  Rows below 16 bytes (NARROW) take single bytes.
__device__ __forceinline__ u32x4 load_bytes(const uint8_t* __restrict__ p, uint32_t n) {  // n < 16
    u32x4 v = 0;
    for (uint32_t k = 0; k < n; k++) {
        const uint32_t b = (uint32_t)p[k] << (8 * (k % 4));
        if (k < 4) v[0] |= b;
        else if (k < 8) v[1] |= b;
        else if (k < 12) v[2] |= b;
        else v[3] |= b;
    }
    return v;
}
template <int KIND, int L, bool NARROW>
__global__ __launch_bounds__(256) void edge_cosine_kernel(const uint8_t* __restrict__ codes, uint64_t stride, uint64_t n_rows, uint32_t dim,
                                                          const uint32_t* __restrict__ eu, const uint32_t* __restrict__ ev, uint64_t n_edges,
                                                          float* __restrict__ cosines) {
    typedef uint32_t any __attribute__((ext_vector_type(4), aligned(1)));
    constexpr uint32_t STEP = L * 16;
    const uint32_t t = threadIdx.x % L;
    for (uint64_t e = (uint64_t)blockIdx.x * (256 / L) + threadIdx.x / L; e < n_edges; e += (uint64_t)gridDim.x * (256 / L)) {
        const uint64_t u = eu[e], v = ev[e];
        const bool ok = u < n_rows && v < n_rows;
        const uint8_t *a = codes + (ok ? u : 0) * stride, *b = codes + (ok ? v : 0) * stride;
        float ab = 0, aa = 0, bb = 0;
        int iab = 0, iaa = 0, ibb = 0;  // 32768 products of at most 2^14: below 2^30
        for (uint32_t c0 = 0; c0 < (ok ? dim : 0); c0 += 4 * STEP) {
            u32x4 x[4], y[4];
            uint32_t skip[4];
#pragma unroll
            for (uint32_t s = 0; s < 4; s++) {
                const uint32_t c = c0 + s * STEP + t * 16;
                x[s] = 0, y[s] = 0, skip[s] = 0;
                if (c0 + s * STEP < dim) {  // the same for all lanes at work
                    if constexpr (NARROW) {
                        if (t == 0) x[s] = load_bytes(a, dim), y[s] = load_bytes(b, dim);
                    } else {
                        const uint32_t at = c < dim - 16 ? c : dim - 16;
                        skip[s] = c - at;
                        x[s] = *reinterpret_cast<const any*>(a + at);
                        y[s] = *reinterpret_cast<const any*>(b + at);
                    }
                }
            }
            if (!NARROW && dim % STEP) {
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int drop = (int)skip[s] - 4 * k;
                        const uint32_t keep = drop >= 4 ? 0u : drop > 0 ? 0xFFFFFFFFu << (8 * drop) : 0xFFFFFFFFu;
                        x[s][k] &= keep, y[s][k] &= keep;
                    }
            }
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (KIND == MDD_I8) {
                        iab = __builtin_amdgcn_sdot4((int)x[s][k], (int)y[s][k], iab, false);
                        iaa = __builtin_amdgcn_sdot4((int)x[s][k], (int)x[s][k], iaa, false);
                        ibb = __builtin_amdgcn_sdot4((int)y[s][k], (int)y[s][k], ibb, false);
                    } else {
                        auto x0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[s][k], false), x1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[s][k], true);
                        auto y0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)y[s][k], false), y1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)y[s][k], true);
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            ab = fmaf(x0[i], y0[i], ab), aa = fmaf(x0[i], x0[i], aa), bb = fmaf(y0[i], y0[i], bb);
                            ab = fmaf(x1[i], y1[i], ab), aa = fmaf(x1[i], x1[i], aa), bb = fmaf(y1[i], y1[i], bb);
                        }
                    }
                }
        }
#pragma unroll
        for (int m = L / 2; m; m >>= 1) {
            if (KIND == MDD_I8) iab += __shfl_xor(iab, m, 64), iaa += __shfl_xor(iaa, m, 64), ibb += __shfl_xor(ibb, m, 64);
            else ab += __shfl_xor(ab, m, 64), aa += __shfl_xor(aa, m, 64), bb += __shfl_xor(bb, m, 64);
        }
        if (KIND == MDD_I8) ab = (float)iab, aa = (float)iaa, bb = (float)ibb;
        // a product of the squares stays below 2^66, and a NaN in a row comes through
        if (t == 0) cosines[e] = !ok || aa == 0.0f || bb == 0.0f ? 0.0f : ab / sqrtf(aa * bb);
    }
}

int check_matrix(const char* who, const char* what, const void* p, int type, uint64_t stride, uint32_t dim) {
    REQUIRE(p, "%s: %s is NULL", who, what);
    REQUIRE(type_bytes(type), "%s: unknown element type %d", who, type);
    REQUIRE(stride >= dim, "%s: row stride %llu of %s is below dim %u", who, (unsigned long long)stride, what, dim);
    REQUIRE(aligned_to(p, type_bytes(type)), "%s: %s is not aligned to its elements", who, what);
    return MDD_OK;
}
#define CHECKED(expr)            \
    do {                         \
        const int rc_ = (expr);  \
        if (rc_) return rc_;     \
    } while (0)

}  // namespace

extern "C" {

uint64_t mdd_embed_ws_bytes(uint64_t n_ids, uint32_t dim) { return pool_ws_bytes(n_ids, dim); }

int mdd_embed(mdd_ctx* ctx, const void* table, int type, uint64_t n_rows, uint64_t row_stride, uint32_t dim, const void* ids,
              int id_bytes, uint64_t n_ids, const uint64_t* offsets, uint64_t n_docs, int mean, float scale, void* out,
              void* ws, uint64_t ws_bytes) {
    const char* who = "mdd_embed";
    REQUIRE(ctx, "%s: ctx is NULL", who);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(type_bytes(type), "%s: unknown element type %d", who, type);
    REQUIRE(id_bytes == 4 || id_bytes == 8, "%s: id_bytes=%d is neither 4 nor 8", who, id_bytes);
    REQUIRE(n_ids < (1ull << 31) && n_rows < (1ull << 32) - 1, "%s: more than 2^31 - 1 ids or 2^32 - 2 table rows", who);
    const uint64_t n_out = offsets ? n_docs : n_ids;
    if (n_out == 0) return MDD_OK;
    REQUIRE(out && aligned_to(out, type_bytes(type)), "%s: out is NULL or not aligned to its elements", who);
    REQUIRE(n_ids == 0 || (ids && aligned_to(ids, id_bytes)), "%s: ids is NULL or not aligned", who);
    if (n_rows) CHECKED(check_matrix(who, "table", table, type, row_stride, dim));
    REQUIRE(row_stride < (1u << 30), "%s: row stride of 2^30 elements or more", who);
    const uint64_t need = offsets && n_rows ? pool_ws_bytes(n_ids, dim) : 0;
    REQUIRE(need == 0 || (ws && aligned_to(ws, 256) && ws_bytes >= need), "%s: workspace of %llu bytes, 256-byte aligned, needed", who,
            (unsigned long long)need);
    ON_DEVICE(ctx);
    if (n_rows == 0 || n_ids == 0) {  // every id is padding
        const uint64_t n = n_out * dim;
        const dim3 grid((unsigned)(n / 256 + 1 < 4096 ? n / 256 + 1 : 4096));
        if (type == MDD_F32) hipLaunchKernelGGL((fill_kernel<uint32_t>), grid, dim3(256), 0, ctx->stream, (uint32_t*)out, n, 0u);
        else hipLaunchKernelGGL((fill_kernel<uint16_t>), grid, dim3(256), 0, ctx->stream, (uint16_t*)out, n, (uint16_t)0);
        HIP_TRY(hipGetLastError());
        return MDD_OK;
    }
    if (!offsets) {
        MDD_FOR_TYPE(type, T, launch_lookup<T>(ctx->stream, (const T*)table, n_rows, row_stride, dim, ids, id_bytes, n_ids, scale, (T*)out));
        HIP_TRY(hipGetLastError());
        return MDD_OK;
    }
    PoolArgs a = {table, n_rows, (uint32_t)(row_stride * type_bytes(type)), dim, lanes_per_row(dim), 1, ids, id_bytes, n_ids, offsets, n_docs, mean, scale, nullptr, piece_log2_for(n_ids), n_pieces_for(n_ids), nullptr,
                  nullptr, nullptr, out};
    if (a.n_pieces) place_parts(a, (uint8_t*)ws);
    MDD_FOR_TYPE(type, T, (launch_pool<T, T, false, false>(ctx->stream, a)));
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

static uint64_t backward_parts(uint64_t n_ids, uint64_t n_docs, uint64_t n_rows, uint32_t dim, uint64_t at[5]) {
    uint64_t o = 0;
    at[0] = o, o += (n_ids > SMALL_SORT ? 4 : 2) * round_up(n_ids * 4, 256);  // keys, values, and the sort's second pair
    at[1] = o, o += round_up(sort_hist_words(n_ids) * 4, 256);
    at[2] = o, o += round_up((n_rows + 1) * 8, 256);          // starts
    at[3] = o, o += round_up(n_docs * 4, 256);                // ids per document
    at[4] = o, o += pool_ws_bytes(n_ids, dim);                // shares of long rows
    return o;
}
uint64_t mdd_embed_backward_ws_bytes(uint64_t n_ids, uint64_t n_docs, uint64_t n_rows, uint32_t dim) {
    uint64_t at[5];
    return backward_parts(n_ids, n_docs, n_rows, dim, at);
}

int mdd_embed_backward(mdd_ctx* ctx, const void* grad, int type, uint64_t grad_stride, uint32_t dim, const void* ids, int id_bytes,
                       uint64_t n_ids, const uint64_t* offsets, uint64_t n_docs, int mean, float scale, void* table_grad,
                       int out_type, uint64_t n_rows, void* ws, uint64_t ws_bytes) {
    const char* who = "mdd_embed_backward";
    REQUIRE(ctx, "%s: ctx is NULL", who);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(type_bytes(type), "%s: unknown element type %d", who, type);
    REQUIRE(out_type == MDD_F32 || out_type == type, "%s: out_type %d is neither MDD_F32 nor the gradient's type", who, out_type);
    REQUIRE(id_bytes == 4 || id_bytes == 8, "%s: id_bytes=%d is neither 4 nor 8", who, id_bytes);
    REQUIRE(n_ids < (1ull << 31) && n_docs < (1ull << 31) && n_rows < (1ull << 31), "%s: 2^31 or more ids, documents or table rows", who);
    if (n_rows == 0) return MDD_OK;
    REQUIRE(table_grad && aligned_to(table_grad, type_bytes(out_type)), "%s: table_grad is NULL or not aligned to its elements", who);
    REQUIRE(n_ids == 0 || (ids && aligned_to(ids, id_bytes)), "%s: ids is NULL or not aligned", who);
    if (!offsets) n_docs = 0;
    const uint64_t n_grad = offsets ? n_docs : n_ids;
    if (n_grad) CHECKED(check_matrix(who, "grad", grad, type, grad_stride, dim));
    REQUIRE(grad_stride < (1u << 30), "%s: row stride of 2^30 elements or more", who);
    uint64_t at[5];
    const uint64_t need = n_ids && n_grad ? backward_parts(n_ids, n_docs, n_rows, dim, at) : 0;
    REQUIRE(need == 0 || (ws && aligned_to(ws, 256) && ws_bytes >= need), "%s: workspace of %llu bytes, 256-byte aligned, needed", who,
            (unsigned long long)need);
    ON_DEVICE(ctx);
    hipStream_t s = ctx->stream;
    if (n_ids == 0 || n_grad == 0) {
        const uint64_t n = n_rows * dim;
        const dim3 grid((unsigned)(n / 256 + 1 < 4096 ? n / 256 + 1 : 4096));
        if (out_type == MDD_F32) hipLaunchKernelGGL((fill_kernel<uint32_t>), grid, dim3(256), 0, s, (uint32_t*)table_grad, n, 0u);
        else hipLaunchKernelGGL((fill_kernel<uint16_t>), grid, dim3(256), 0, s, (uint16_t*)table_grad, n, (uint16_t)0);
        HIP_TRY(hipGetLastError());
        return MDD_OK;
    }
    uint8_t* base = (uint8_t*)ws;
    uint32_t *key = (uint32_t*)(base + at[0]), *val = key + round_up(n_ids, 64), *key2 = val + round_up(n_ids, 64), *val2 = key2 + round_up(n_ids, 64);
    uint64_t* start = (uint64_t*)(base + at[2]);
    uint32_t* count = mean && offsets ? (uint32_t*)(base + at[3]) : nullptr;
    if (count) hipLaunchKernelGGL((fill_kernel<uint32_t>), dim3((unsigned)(n_docs / 256 + 1 < 4096 ? n_docs / 256 + 1 : 4096)), dim3(256), 0, s, count, n_docs, 0u);
    const GradIds g = {ids, id_bytes, n_ids, n_rows, offsets, n_docs, count};
    const int bits = bits_of(n_rows);
    const dim3 per_id(grid_for(n_ids, 256));
    if (n_ids <= SMALL_SORT && (!offsets || n_ids <= 1024)) {
        // one launch less; but finding the document of each position is slow work for a single block (8000 ids in 80 documents:
        // a gradient of 51 us made on the way in, 39 with a launch of their own; 2000 ids the same either way)
        hipLaunchKernelGGL(small_sort_kernel<true>, dim3(1), dim3(1024), 0, s, key, val, (uint32_t)n_ids, 0, bits, g);
    } else {
        hipLaunchKernelGGL(grad_keys_kernel, per_id, dim3(256), 0, s, g, key, val);
        if (n_ids <= SMALL_SORT) hipLaunchKernelGGL(small_sort_kernel<false>, dim3(1), dim3(1024), 0, s, key, val, (uint32_t)n_ids, 0, bits, g);
        else sort_pairs(s, key, val, key2, val2, n_ids, bits, (uint32_t*)(base + at[1]));
    }
    hipLaunchKernelGGL(grad_starts_kernel, dim3(grid_for(n_rows + 1, 256)), dim3(256), 0, s, key, (uint32_t)n_ids, n_rows, start);
    // the sums themselves are a lookup: table rows are the documents, the sorted positions their ids, grad the table.
    // 262144 x 1024 in bf16 into 64000 rows, 800 MB read and written: 199 us with the sort, 219 through the caches; gradients
    // that fit the last-level cache come out of it (262144 x 256: 82 us, 98 past it)
    const bool once = !offsets && n_grad * dim * type_bytes(type) > LAST_LEVEL;  // with documents a row is read for each of its ids
    PoolArgs a = {grad, n_grad, (uint32_t)(grad_stride * type_bytes(type)), dim, lanes_per_row(dim), 1, val, 4, n_ids, start, n_rows, 0, scale, count, piece_log2_for(n_ids), n_pieces_for(n_ids),
                  nullptr, nullptr, nullptr, table_grad};
    if (a.n_pieces) place_parts(a, base + at[4]);
    MDD_FOR_TYPE(type, T, {
        auto run = [&](auto* out) {
            typedef std::remove_pointer_t<decltype(out)> O;
            count ? launch_pool<T, O, true, false>(s, a) : once ? launch_pool<T, O, false, true>(s, a) : launch_pool<T, O, false, false>(s, a);
        };
        if (out_type == MDD_F32) run((float*)nullptr);
        else run((T*)nullptr);
    });
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

int mdd_rms_norm(mdd_ctx* ctx, const void* x, int type, uint64_t x_stride, const void* residual, uint64_t residual_stride,
                 const void* weight, float eps, uint64_t n_rows, uint32_t dim, void* y, void* sum_out, float* rstd) {
    const char* who = "mdd_rms_norm";
    REQUIRE(ctx, "%s: ctx is NULL", who);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(eps >= 0.0f, "%s: eps=%g is not a number >= 0", who, (double)eps);
    REQUIRE(type_bytes(type), "%s: unknown element type %d", who, type);
    if (n_rows == 0) return MDD_OK;
    CHECKED(check_matrix(who, "x", x, type, x_stride, dim));
    if (residual) CHECKED(check_matrix(who, "residual", residual, type, residual_stride, dim));
    if (weight) CHECKED(check_matrix(who, "weight", weight, type, dim, dim));
    CHECKED(check_matrix(who, "y", y, type, dim, dim));
    REQUIRE(!sum_out || aligned_to(sum_out, type_bytes(type)), "%s: sum_out is not aligned to its elements", who);
    REQUIRE(!rstd || aligned_to(rstd, 4), "%s: rstd is not aligned", who);
    const bool once = n_rows * dim * type_bytes(type) * (2 + (residual != nullptr) + (sum_out != nullptr)) > LAST_LEVEL;
    ON_DEVICE(ctx);
    MDD_FOR_TYPE(type, T, {
        for_width(dim, false, [&](auto nc, auto l, auto narrow) {
            auto kernel = once ? norm_kernel<T, nc.value, l.value, narrow.value, true> : norm_kernel<T, nc.value, l.value, narrow.value, false>;
            hipLaunchKernelGGL(kernel, row_grid(n_rows, l.value), dim3(l.value == 1024 ? 1024 : 256), 0, ctx->stream,
                               (const T*)x, x_stride, (const T*)residual, residual_stride, (const T*)weight, eps, n_rows, dim, (T*)y, (T*)sum_out, rstd);
        });
    });
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

int mdd_rms_norm_q8(mdd_ctx* ctx, const void* x, int type, uint64_t x_stride, const void* residual, uint64_t residual_stride,
                    const void* weight, float eps, uint64_t n_rows, uint32_t dim, int kind, void* codes, float* scales, void* sum_out) {
    const char* who = "mdd_rms_norm_q8";
    REQUIRE(ctx, "%s: ctx is NULL", who);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(eps >= 0.0f, "%s: eps=%g is not a number >= 0", who, (double)eps);
    REQUIRE(type_bytes(type), "%s: unknown element type %d", who, type);
    REQUIRE(kind == MDD_I8 || kind == MDD_E4M3, "%s: unknown 8-bit kind %d", who, kind);
    if (n_rows == 0) return MDD_OK;
    CHECKED(check_matrix(who, "x", x, type, x_stride, dim));
    if (residual) CHECKED(check_matrix(who, "residual", residual, type, residual_stride, dim));
    if (weight) CHECKED(check_matrix(who, "weight", weight, type, dim, dim));
    REQUIRE(codes && scales && aligned_to(scales, 4), "%s: NULL buffer, or scales not aligned", who);
    REQUIRE(!sum_out || aligned_to(sum_out, type_bytes(type)), "%s: sum_out is not aligned to its elements", who);
    const bool once = n_rows * dim * (type_bytes(type) * (1 + (residual != nullptr) + (sum_out != nullptr)) + 1) > LAST_LEVEL;
    ON_DEVICE(ctx);
    MDD_FOR_TYPE(type, T, {
        for_width(dim, false, [&](auto nc, auto l, auto narrow) {
            auto kernel = kind == MDD_I8 ? (once ? norm_q8_kernel<T, nc.value, l.value, MDD_I8, narrow.value, true> : norm_q8_kernel<T, nc.value, l.value, MDD_I8, narrow.value, false>)
                                         : (once ? norm_q8_kernel<T, nc.value, l.value, MDD_E4M3, narrow.value, true> : norm_q8_kernel<T, nc.value, l.value, MDD_E4M3, narrow.value, false>);
            hipLaunchKernelGGL(kernel, row_grid(n_rows, l.value), dim3(l.value == 1024 ? 1024 : 256), 0, ctx->stream, (const T*)x, x_stride,
                               (const T*)residual, residual_stride, (const T*)weight, eps, n_rows, dim, (uint8_t*)codes, scales, (T*)sum_out);
        });
    });
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

uint64_t mdd_rms_norm_backward_ws_bytes(uint64_t n_rows, uint32_t dim) { return round_up((uint64_t)backward_blocks(n_rows, dim) * dim * 4, 256); }

int mdd_rms_norm_backward(mdd_ctx* ctx, const void* grad, int type, uint64_t grad_stride, const void* h, uint64_t h_stride,
                          const void* grad_sum, uint64_t grad_sum_stride, const void* weight, const float* rstd,
                          uint64_t n_rows, uint32_t dim, void* x_grad, float* weight_grad, void* ws, uint64_t ws_bytes) {
    const char* who = "mdd_rms_norm_backward";
    REQUIRE(ctx, "%s: ctx is NULL", who);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(type_bytes(type), "%s: unknown element type %d", who, type);
    REQUIRE(!weight_grad || aligned_to(weight_grad, 4), "%s: weight_grad is not aligned", who);
    if (n_rows) {
        CHECKED(check_matrix(who, "grad", grad, type, grad_stride, dim));
        CHECKED(check_matrix(who, "h", h, type, h_stride, dim));
        if (grad_sum) CHECKED(check_matrix(who, "grad_sum", grad_sum, type, grad_sum_stride, dim));
        if (weight) CHECKED(check_matrix(who, "weight", weight, type, dim, dim));
        CHECKED(check_matrix(who, "x_grad", x_grad, type, dim, dim));
        REQUIRE(rstd && aligned_to(rstd, 4), "%s: rstd is NULL or not aligned", who);
    }
    const uint32_t blocks = backward_blocks(n_rows, dim);
    const uint64_t need = mdd_rms_norm_backward_ws_bytes(n_rows, dim);
    REQUIRE(!weight_grad || n_rows == 0 || (ws && aligned_to(ws, 256) && ws_bytes >= need), "%s: workspace of %llu bytes, 256-byte aligned, needed", who,
            (unsigned long long)need);
    ON_DEVICE(ctx);
    if (n_rows == 0) {
        if (weight_grad) hipLaunchKernelGGL((fill_kernel<float>), dim3((dim + 255) / 256), dim3(256), 0, ctx->stream, weight_grad, (uint64_t)dim, 0.0f);
        HIP_TRY(hipGetLastError());
        return MDD_OK;
    }
    float* part = weight_grad ? (float*)ws : nullptr;
    MDD_FOR_TYPE(type, T, {
        for_width(dim, true, [&](auto nc, auto l, auto narrow) {
            hipLaunchKernelGGL((norm_backward_kernel<T, nc.value, l.value, narrow.value>), dim3(blocks), dim3(l.value == 1024 ? 1024 : 256), 0, ctx->stream, (const T*)grad,
                               grad_stride, (const T*)h, h_stride, (const T*)grad_sum, grad_sum_stride, (const T*)weight, rstd, n_rows, dim, (T*)x_grad, part);
        });
    });
    if (weight_grad)
        hipLaunchKernelGGL(weight_grad_kernel, dim3((dim + 63) / 64), dim3(1024), 0, ctx->stream, part, blocks, dim, weight_grad);
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

int mdd_edge_cosines(mdd_ctx* ctx, const void* codes, int kind, uint64_t row_stride, uint64_t n_rows, uint32_t dim,
                     const uint32_t* edge_u, const uint32_t* edge_v, uint64_t n_edges, float* cosines) {
    const char* who = "mdd_edge_cosines";
    REQUIRE(ctx, "%s: ctx is NULL", who);
    REQUIRE(kind == MDD_I8 || kind == MDD_E4M3, "%s: unknown 8-bit kind %d", who, kind);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(row_stride >= dim, "%s: row stride below dim", who);
    if (n_edges == 0) return MDD_OK;
    REQUIRE((codes || n_rows == 0) && edge_u && edge_v && cosines, "%s: NULL buffer", who);
    ON_DEVICE(ctx);
    auto launch = [&](auto lanes, auto narrow) {
        constexpr int L = decltype(lanes)::value;
        const uint64_t want = (n_edges * L + 255) / 256, cap = (uint64_t)ctx->cus * 64;
        auto kernel = kind == MDD_I8 ? edge_cosine_kernel<MDD_I8, L, decltype(narrow)::value> : edge_cosine_kernel<MDD_E4M3, L, decltype(narrow)::value>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(want < cap ? want : cap)), dim3(256), 0, ctx->stream, (const uint8_t*)codes, row_stride, n_rows, dim, edge_u,
                           edge_v, n_edges, cosines);
    };
    if (dim < 16) launch(std::integral_constant<int, 4>(), std::true_type());
    else if (dim <= 64) launch(std::integral_constant<int, 4>(), std::false_type());
    else if (dim <= 128) launch(std::integral_constant<int, 8>(), std::false_type());
    else launch(std::integral_constant<int, 16>(), std::false_type());
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

uint64_t mdd_sort_edges_ws_bytes(uint64_t n_edges) {
    return n_edges <= SMALL_SORT ? 0 : 2 * round_up(n_edges * 4, 256) + round_up(sort_hist_words(n_edges) * 4, 256);
}

int mdd_sort_edges(mdd_ctx* ctx, uint32_t* edge_u, uint32_t* edge_v, uint64_t n_edges, uint64_t n_docs, void* ws, uint64_t ws_bytes) {
    const char* who = "mdd_sort_edges";
    REQUIRE(ctx, "%s: ctx is NULL", who);
    REQUIRE(n_edges < (1ull << 31) && n_docs <= 0xFFFFFFFFull, "%s: 2^31 or more edges, or 2^32 or more documents", who);
    if (n_edges <= 1) return MDD_OK;
    REQUIRE(edge_u && edge_v, "%s: NULL buffer", who);
    const uint64_t need = mdd_sort_edges_ws_bytes(n_edges);
    REQUIRE(need == 0 || (ws && aligned_to(ws, 256) && ws_bytes >= need), "%s: workspace of %llu bytes, 256-byte aligned, needed", who,
            (unsigned long long)need);
    ON_DEVICE(ctx);
    const int bits = bits_of(n_docs ? n_docs - 1 : 0);
    uint32_t *u = edge_u, *v = edge_v, *v2 = (uint32_t*)ws, *u2 = v2 + round_up(n_edges, 64), *hist = u2 + round_up(n_edges, 64);
    if (n_edges <= SMALL_SORT) {
        hipLaunchKernelGGL(small_sort_kernel<false>, dim3(1), dim3(1024), 0, ctx->stream, edge_u, edge_v, (uint32_t)n_edges, bits, bits, GradIds());
        HIP_TRY(hipGetLastError());
        return MDD_OK;
    }
    // by the second column, then stably by the first; the passes of both together are even in number, so the result ends up
    // in the caller's arrays
    sort_pairs(ctx->stream, v, u, v2, u2, n_edges, bits, hist);
    sort_pairs(ctx->stream, u, v, u2, v2, n_edges, bits, hist);
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

}  // extern "C"
