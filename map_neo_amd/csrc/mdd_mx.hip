// Microscaled 4-bit matrices: quantisation, product, near pairs.  Declarations, formats and contracts: include/mdd.h.
#include "mdd_vec.h"

#include <type_traits>

using namespace mddi;

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr uint32_t TILE = 2048, STILE = 128;  // bytes of a 32 x 128 tile: codes, scales

// ------------------------------------------------------------------------------------------------ quantisation
// A wave takes half a tile: sixteen lanes side by side read 128 columns of a row, four lanes share a block of 32, and four times
// four rows are in flight.  The lanes' maxima meet across the four, each converts its eight elements to a word, and a
// transposition among the four lets each store the 16 bytes of a block whole.  Bound by HBM: the matrix is read once, a bit
// more than half a byte per element is written -- 262144 x 1024 in bf16 in 125 us, 5.4 TB/s, 45000 x 768 in 15. A thread a
// block of 32 columns, whose loads lie 64 bytes apart, took 155 and 26 us, a wave a tile, all of which load at once and then
// store at once, 130 and 25.
__device__ __forceinline__ uint32_t swap1(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true); }  // lane ^ 1
__device__ __forceinline__ uint32_t swap2(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true); }  // lane ^ 2
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, uint64_t stride, uint64_t n_rows, uint32_t dim,
                                                          uint64_t n_halves, uint32_t col_tiles, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
    const uint32_t lane = lane_id(), q = lane % 4, kb = lane / 4 % 4, g = lane / 16;
    for (uint64_t half = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64; half < n_halves; half += (uint64_t)gridDim.x * 4) {
        const uint64_t rt = half / (2 * col_tiles);
        const uint32_t in = (uint32_t)(half - rt * (2 * col_tiles)), up = in >= col_tiles ? 16 : 0, ct = up ? in - col_tiles : in, col = ct * 128 + lane % 16 * 8;
        const uint64_t tile = rt * col_tiles + ct, row0 = rt * 32 + up + g;  // rows row0, row0 + 4, 8, 12
        typename vec8<T>::raw raw[4];
        if (rt * 32 + up + 16 <= n_rows && ct * 128 + 128 <= dim) {  // four loads without a branch
#pragma unroll
            for (int i = 0; i < 4; i++) raw[i] = *reinterpret_cast<const typename vec8<T>::raw_any*>(x + (row0 + i * 4) * stride + col);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                raw[i] = (T)0.0f;
                if (row0 + i * 4 < n_rows && col < dim) raw[i] = load8_raw<T>(x + (row0 + i * 4) * stride + col, dim - col);
            }
        }
        uint32_t w[4], sb[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f32x8 v = __builtin_convertvector(raw[i], f32x8);
            uint32_t big = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint32_t m = __float_as_uint(v[k]) & 0x7FFFFFFFu;
                big = m > big ? m : big;
            }
            uint32_t o = swap1(big);
            big = o > big ? o : big;
            o = swap2(big);
            big = o > big ? o : big;
            // biased exponent of the largest, less 2; subnormal and zero blocks stop at 2^-127
            const int e = (int)(big >> 23) - 127 - 2, sc = e > -127 ? e : -127;
            const bool bad = big >= 0x7F800000u;
            const float scale = sc > -127 ? __uint_as_float((uint32_t)(sc + 127) << 23) : 0x1p-127f;
            // divides by the scale, rounds to the nearest, ties to even, and stops at 6
            uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], scale, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
            w[i] = bad ? 0u : c;
            sb[i] = row0 + i * 4 >= n_rows || ct * 128 + kb * 32 >= dim ? 127u : bad ? 255u : (uint32_t)(sc + 127);
        }
#pragma unroll
        for (int k = 0; k < 4; k += 2) {  // lane q of the four takes row q
            const uint32_t o = swap1(q & 1 ? w[k] : w[k + 1]);
            w[k] = q & 1 ? o : w[k];
            w[k + 1] = q & 1 ? w[k + 1] : o;
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t o = swap2(q & 2 ? w[k] : w[k + 2]);
            w[k] = q & 2 ? o : w[k];
            w[k + 2] = q & 2 ? w[k + 2] : o;
        }
        const uint32_t r = up + q * 4 + g, s0 = q & 1 ? sb[1] : sb[0], s1 = q & 1 ? sb[3] : sb[2];
        const u32x4 p = {w[0], w[1], w[2], w[3]};
        *reinterpret_cast<u32x4*>(codes + tile * TILE + kb * 512 + r * 16) = p;
        scales[tile * STILE + (kb & 1) * 64 + r * 2 + (kb >> 1)] = (uint8_t)(q & 2 ? s1 : s0);
    }
}

// ------------------------------------------------------------------------------------------------ product
// One matrix instruction multiplies 32 x 64 by 64 x 32 (v_mfma_scale_f32_32x32x64_f8f6f4): lane l holds row l % 32 and the 32
// columns of block l / 32, 16 bytes and one scale byte -- which is why the packed tile stores [block][row][16 bytes]: a
// fragment is 1 KB in lane order, read from memory or from LDS without a stride.  First operand: rows of B, second: rows
// of A, so that a lane ends up with four neighbouring columns of C in one row.
__device__ __forceinline__ f32x16 mma(i32x4 b, int sb, i32x4 a, int sa, f32x16 c, int half) {
    const i32x8 b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0}, a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
    if (half) return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b8, a8, c, 4, 4, 1, sb, 1, sa);
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b8, a8, c, 4, 4, 0, sb, 0, sa);
}

template <typename O>
__device__ __forceinline__ void store_quad(O* __restrict__ p, uint32_t n, float a, float b, float c, float d) {
    typedef O quad __attribute__((ext_vector_type(4)));
    typedef O quad_any __attribute__((ext_vector_type(4), aligned(sizeof(O))));
    const quad q = {(O)a, (O)b, (O)c, (O)d};
    if (n >= 4) {
        *reinterpret_cast<quad_any*>(p) = q;
    } else {
        for (uint32_t k = 0; k < 3; k++)
            if (k < n) p[k] = q[k];
    }
}

// Few rows of A, or few of both: every wave streams one row tile of B from memory and multiplies it with FM row tiles of A (of a
// group of four by blockIdx.y), whose fragments come out of the caches.  Bound by reading B: one row against 262144 x 1024 in
// 24 us, 142 MB at 5.9 TB/s (the last-level cache holds half).  SPLIT waves share a tile's columns where there are too few tiles
// to fill the chip; their sums are joined in LDS in wave order.  With few rows of B it is A that streams: then the two change
// places, and a result goes to where its row and column say (swapped).
template <typename O, int FM, int SPLIT>
__global__ __launch_bounds__(256) void mx_skinny_kernel(const uint8_t* __restrict__ ac, const uint8_t* __restrict__ as, uint64_t m, uint32_t a_tiles,
                                                        const uint8_t* __restrict__ bc, const uint8_t* __restrict__ bs, uint64_t n, uint64_t b_tiles,
                                                        uint32_t col_tiles, float alpha, O* __restrict__ c, uint64_t cs, bool swapped) {
    constexpr int U = FM == 1 ? 4 : 2;  // column tiles in flight
    __shared__ float join[SPLIT > 1 ? (SPLIT - 1) * FM * 16 * 64 : 1];
    const uint32_t lane = lane_id(), wave = threadIdx.x / 64, part = wave % SPLIT;
    const uint64_t tile = (uint64_t)blockIdx.x * (4 / SPLIT) + wave / SPLIT;
    const uint64_t first = (uint64_t)blockIdx.y * FM, here = a_tiles - first;  // row tiles of A: from which on, and how many there are
    f32x16 acc[FM];
#pragma unroll
    for (int f = 0; f < FM; f++) acc[f] = 0.0f;
    if (tile < b_tiles) {
        const uint8_t *bp = bc + tile * col_tiles * TILE + lane * 16, *sp = bs + tile * col_tiles * STILE + lane * 2;
        const uint8_t *ap = ac + first * col_tiles * TILE + lane * 16, *tp = as + first * col_tiles * STILE + lane * 2;
#pragma unroll 1
        for (uint32_t k0 = part * U; k0 < col_tiles; k0 += SPLIT * U) {
            i32x4 b[U][2], a[U][FM][2];
            int sb[U], sa[U][FM];
#pragma unroll
            for (int u = 0; u < U; u++) {
                // past the last column tile: any tile's bytes, dropped below
                const uint64_t k = k0 + u < col_tiles ? k0 + u : col_tiles - 1;
                b[u][0] = *reinterpret_cast<const i32x4*>(bp + k * TILE);
                b[u][1] = *reinterpret_cast<const i32x4*>(bp + k * TILE + 1024);
                sb[u] = *reinterpret_cast<const uint16_t*>(sp + k * STILE);
#pragma unroll
                for (int f = 0; f < FM; f++) {
                    const uint64_t at = ((uint64_t)f < here ? f : here - 1) * col_tiles + k;
                    a[u][f][0] = *reinterpret_cast<const i32x4*>(ap + at * TILE);
                    a[u][f][1] = *reinterpret_cast<const i32x4*>(ap + at * TILE + 1024);
                    sa[u][f] = *reinterpret_cast<const uint16_t*>(tp + at * STILE);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (k0 + u < col_tiles)
#pragma unroll
                    for (int f = 0; f < FM; f++) {
                        acc[f] = mma(b[u][0], sb[u], a[u][f][0], sa[u][f], acc[f], 0);
                        acc[f] = mma(b[u][1], sb[u], a[u][f][1], sa[u][f], acc[f], 1);
                    }
        }
    }
    if (SPLIT > 1) {
        if (part) {
#pragma unroll
            for (int f = 0; f < FM; f++)
#pragma unroll
                for (int i = 0; i < 16; i++) join[(((part - 1) * FM + f) * 16 + i) * 64 + lane] = acc[f][i];
        }
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int s = 0; s < SPLIT - 1; s++)
#pragma unroll
            for (int f = 0; f < FM; f++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[f][i] += join[((s * FM + f) * 16 + i) * 64 + lane];
    }
    if (tile >= b_tiles) return;
#pragma unroll
    for (int f = 0; f < FM; f++) {
        const uint64_t row = (first + f) * 32 + lane % 32;
        if (row >= m) continue;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint64_t col = tile * 32 + q * 8 + lane / 32 * 4;
            if (swapped) {
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (col + k < n) c[(col + k) * cs + row] = (O)(alpha * acc[f][q * 4 + k]);
            } else if (col < n)
                store_quad<O>(c + row * cs + col, (uint32_t)(n - col < 4 ? n - col : 4), alpha * acc[f][q * 4], alpha * acc[f][q * 4 + 1],
                              alpha * acc[f][q * 4 + 2], alpha * acc[f][q * 4 + 3]);
        }
    }
}

// Tiled product.  A block of WR x WC waves computes (WR * FM * 32) x (WC * FN * 32) of C and walks a list of such tiles.  Column
// tiles (128 columns: a step) go from memory straight into LDS, three buffers in rotation, in one stream of steps that runs
// on across the tiles of the list: while a tile's results leave, the next tile's first steps are landing.  A step is two
// halves of 64 columns.  The fragments of a half are read from LDS while the half before is multiplied:
//     multiply half 0 of step s, and between the products: read half 1 of step s
//     wait for step s + 1, barrier
//     multiply half 1 of step s, and between them: read half 0 of step s + 1, request step s + 3 into the buffer of step s
// so a load has two steps to arrive, a step needs one barrier, and neither LDS nor memory latency nor the issue of loads stands
// before the matrix unit.  8192 x 16384 x 8192: 4.2 PFLOP/s on random numbers, 5.5 on zeros, of 10 that the units could do at 2.4 GHz.
// Two things keep it there.  The units are busy 46 % of the cycles (8192 x 32768 x 2048; 44 % among pairs), on zeros as well: a step
// multiplies for 1024 cycles and takes 96 KB of fragments and 34 KB of arriving tiles through an LDS of 128 bytes a cycle, 1040
// cycles, and the two do not overlap fully.  And the card lowers its clock with what switches: 1.8 GHz on random numbers, 2.26 on zeros.
// (Four waves of 128 x 128, which read a third less from LDS, do the same 4.1 but have nothing to overlap a tile's end with: 2048
// columns 186 us against 147.)
template <int WR_, int WC_, int FM_, int FN_>
struct Block {
    static constexpr int WR = WR_, WC = WC_, FM = FM_, FN = FN_;
    static constexpr int WAVES = WR * WC, TA = WR * FM, TB = WC * FN, TILES = TA + TB, PER_WAVE = TILES / WAVES;
    static constexpr uint32_t STAGE = TILES * (TILE + STILE), LDS = 3 * STAGE, OUT = 4096;  // OUT: a wave's room to turn results round
    static constexpr int LOADS = PER_WAVE * 2 + 1;  // per wave and step: two halves of each of its tiles, and their scales
    static_assert(TILES == 2 * WAVES, "every wave loads two tiles, and their scales in one instruction of four bytes a lane");
};
// 256 x 256, 8 waves, one block a CU.  (128 x 128 by 4 waves, two blocks a CU, is no quicker even for a few tiles, whose steps then
// have too few products to hide anything: 200 x 129 x 8192 64 us against 52, 45000 x 384 near pairs 447 against 220.)
using Tiles = Block<4, 2, 2, 4>;

// 16 (4) bytes of every lane from its own address to LDS, lane after lane from l on
__device__ __forceinline__ void to_lds(const uint8_t* g, uint8_t* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)g, (__attribute__((address_space(3))) uint32_t*)l, 16, 0, 0);
}
__device__ __forceinline__ void to_lds4(const uint8_t* g, uint8_t* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)g, (__attribute__((address_space(3))) uint32_t*)l, 4, 0, 0);
}
// Waits by the builtin, not by a statement in assembly: the compiler then knows that nothing before is left to wait for.
// (vmcnt bits 0-3 and 14-15, expcnt 4-6, lgkmcnt 8-11)
template <int N>
__device__ __forceinline__ void wait_memory() {  // at most N of this wave's memory operations outstanding
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0xF70);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {  // this wave's LDS reads done
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
}

// The compiler would move a half's products down behind the barrier, next to their use in the other half's; an empty
// statement that takes the results keeps them before it, where they cover the LDS reads and the wait.
template <int FM, int FN>
__device__ __forceinline__ void keep_here(f32x16 (&acc)[FM][FN]) {
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) asm volatile("" : "+v"(acc[i][j]));
}

struct Packed {
    const uint8_t *codes, *scales;
    uint32_t tiles;  // row tiles
};
struct Place {
    uint32_t i0, j0;  // first row tile of A and of B; the same in every lane
    bool valid;
};
__device__ __forceinline__ Place place_at(uint32_t i0, uint32_t j0) { return {(uint32_t)__builtin_amdgcn_readfirstlane(i0), (uint32_t)__builtin_amdgcn_readfirstlane(j0), true}; }
struct Cursor {  // of a block's walk through the list: the round that comes next, and the band of the last tile
    uint32_t first = 0, band = 0;
};
constexpr uint64_t MAX_TILES = 1ull << 31;  // of a list

// next(cursor) is the block's next tile (valid = false: the list is done).  begin(place) is called before a tile's steps and
// finish(place, acc) takes its results; it returns whether it has issued at least STORES memory operations.
template <typename B, int STORES, typename F, typename I, typename G>
__device__ __forceinline__ void mx_stream(const Packed a, const Packed b, uint32_t col_tiles, uint8_t* lds, F&& next, I&& begin, G&& finish) {
    constexpr int FM = B::FM, FN = B::FN;
    const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wr = wave / B::WC, wc = wave % B::WC;
    Cursor req_cursor, cursor;
    Place req = next(req_cursor), cur = next(cursor);
    if (!cur.valid) return;
    uint32_t req_k = 0, req_buf = 0;
    Place ahead = {0, 0, false};  // the tile last turned to
    const uint8_t *src[B::PER_WAVE], *ssrc;
    auto aim = [&]() {  // this wave's share: PER_WAVE row tiles.  Tiles past the end repeat the last one; their results are not used
        auto at = [&](uint32_t t, const uint8_t* pa, const uint8_t* pb, uint32_t bytes) {
            const bool is_a = t < (uint32_t)B::TA;
            const uint32_t rt = is_a ? req.i0 + t : req.j0 + t - B::TA, last = (is_a ? a.tiles : b.tiles) - 1;
            return (is_a ? pa : pb) + (uint64_t)(rt < last ? rt : last) * col_tiles * bytes;
        };
#pragma unroll
        for (int i = 0; i < B::PER_WAVE; i++) src[i] = at(wave * B::PER_WAVE + i, a.codes, b.codes, TILE);
        ssrc = at(wave * B::PER_WAVE + lane / 32, a.scales, b.scales, STILE) + lane % 32 * 4;
    };
    aim();
    // A request is one load instruction of 1 KB at a time, `item` 0 .. LOADS - 1, so that it can be strewn among the products.
    const uint8_t *from[B::PER_WAVE], *sfrom;
    uint8_t* into;
    auto turn_to_next = [&]() {  // the stream's next step.  Behind the list's end the last tile again: never used, always there
#pragma unroll
        for (int i = 0; i < B::PER_WAVE; i++) from[i] = src[i] + (uint64_t)req_k * TILE;
        sfrom = ssrc + (uint64_t)req_k * STILE;
        into = lds + req_buf * B::STAGE;
        req_buf = req_buf == 2 ? 0 : req_buf + 1;
        if (++req_k == col_tiles) {
            req_k = 0;
            ahead = next(req_cursor);
            if (ahead.valid) {
                req = ahead;
                aim();
            }
        }
    };
    auto request = [&](int item) {
        if (item < 2 * B::PER_WAVE)
            to_lds(from[item / 2] + item % 2 * 1024 + lane * 16, into + (wave * B::PER_WAVE + item / 2) * TILE + item % 2 * 1024);
        else
            to_lds4(sfrom, into + B::TILES * TILE + wave * B::PER_WAVE * STILE);
    };
    i32x4 fa[2][FM], fb[2][FN];
    int xa[FM], xb[FN], ya[FM], yb[FN];  // a step's scales, both halves in one register; the next step's
    auto read_one = [&](uint32_t buf, int h, int item) {  // fragments 0 .. FM + FN - 1
        const uint8_t* l = lds + buf * B::STAGE + h * 1024 + lane * 16;
        if (item < FM) fa[h][item] = *reinterpret_cast<const i32x4*>(l + (wr * FM + item) * TILE);
        else fb[h][item - FM] = *reinterpret_cast<const i32x4*>(l + (B::TA + wc * FN + item - FM) * TILE);
    };
    auto read_scales = [&](uint32_t buf) {
        const uint8_t* s = lds + buf * B::STAGE + B::TILES * TILE + lane * 2;
#pragma unroll
        for (int i = 0; i < FM; i++) ya[i] = *reinterpret_cast<const uint16_t*>(s + (wr * FM + i) * STILE);
#pragma unroll
        for (int j = 0; j < FN; j++) yb[j] = *reinterpret_cast<const uint16_t*>(s + (B::TA + wc * FN + j) * STILE);
    };
    f32x16 acc[FM][FN];
    auto multiply = [&](int h, int x, bool fresh) {  // fresh: the tile's first product, to nothing added
        const int i = x / FN, j = x % FN;
        const f32x16 none = 0.0f;
        acc[i][j] = mma(fb[h][j], xb[j], fa[h][i], xa[i], fresh ? none : acc[i][j], h);
    };
    auto take_scales = [&]() {
#pragma unroll
        for (int i = 0; i < FM; i++) xa[i] = ya[i];
#pragma unroll
        for (int j = 0; j < FN; j++) xb[j] = yb[j];
    };
    constexpr int PRODUCTS = FM * FN, READS = FM + FN, ITEMS = READS + 1 + B::LOADS;
    constexpr int A_EACH = (READS + PRODUCTS - 3) / (PRODUCTS - 2), B_EACH = (ITEMS + PRODUCTS - 1) / PRODUCTS;

#pragma unroll 1
    for (int r = 0; r < 3; r++) {
        turn_to_next();
#pragma unroll
        for (int i = 0; i < B::LOADS; i++) request(i);
    }
    wait_memory<2 * B::LOADS>();
    __builtin_amdgcn_s_barrier();
    uint32_t buf = 0;
    read_scales(0);
#pragma unroll
    for (int i = 0; i < READS; i++) read_one(0, 0, i);
    take_scales();
    int behind = 0;  // steps for which finish's operations are younger than the loads waited for
    auto step = [&](auto fresh) {
        turn_to_next();
        // a product keeps the matrix unit busy for 32 cycles: what else a half has to issue goes between them
#pragma unroll
        for (int x = 0; x < PRODUCTS; x++) {
            multiply(0, x, decltype(fresh)::value);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = x * A_EACH; i < (x + 1) * A_EACH && i < READS; i++) read_one(buf, 1, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        keep_here(acc);
        // step s + 1 has landed when only younger operations are left: the loads of step s + 2, and for two steps after a tile
        // the stores of its results.  And this wave has read all it wants of the buffer of step s, which is requested anew
        // behind the barrier.
        wait_lds();
        if (behind > 0) wait_memory<B::LOADS + STORES>();
        else wait_memory<B::LOADS>();
        __builtin_amdgcn_s_barrier();
        behind--;
        buf = buf == 2 ? 0 : buf + 1;  // behind the last step: whatever the buffer holds, not used
#pragma unroll
        for (int x = 0; x < PRODUCTS; x++) {
            multiply(1, x, false);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = x * B_EACH; i < (x + 1) * B_EACH && i < ITEMS; i++) {
                if (i < READS) read_one(buf, 0, i);
                else if (i == READS) read_scales(buf);
                else request(i - READS - 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        keep_here(acc);
        __builtin_amdgcn_sched_barrier(0);  // the reads have had the products' time to arrive
        take_scales();
    };
    while (cur.valid) {
        begin(cur);
        wait_lds();
        step(std::true_type());
#pragma unroll 1
        for (uint32_t k = 1; k < col_tiles; k++) step(std::false_type());
        behind = finish(cur, acc) ? 2 : 0;
        // requests are three steps ahead: with four steps a tile or more, the tile turned to last is the one after this
        if (col_tiles >= 4) cur = ahead;
        else cur = next(cursor);
    }
    wait_memory<0>();  // loads into LDS do not outlive the block
}

// Work order.  An XCD gets a run of consecutive tiles of the list, and the list walks eight block rows at a time down the
// columns: the 32 blocks that an XCD runs together share 8 + 4 tiles out of its L2.
// Position in the list of this block's round that begins at `first`; `total` when there is none
__device__ __forceinline__ uint32_t list_place(uint32_t first, uint32_t total) {
    if (first >= total || blockIdx.x >= total - first) return total;
    return first + xcd_order(blockIdx.x, total - first < gridDim.x ? total - first : gridDim.x);
}

// Results leave through LDS: a lane holds four neighbouring columns of one row, which alone would be 32 rows of 16 bytes per
// store; turned round in 4 KB of LDS (32 rows x 128 bytes, 16-byte pieces exchanged by row against bank conflicts) eight lanes
// write 128 bytes of a row: 8192 x 16384 x 128 in bf16, all result, 117 -> 45 us.
template <typename O, typename B>
__global__ __launch_bounds__(B::WAVES * 64) void mx_matmul_kernel(const Packed a, uint64_t m, const Packed b, uint64_t n, uint32_t col_tiles, float alpha,
                                                                  O* __restrict__ c, uint64_t cs) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    constexpr int JO = 4 / sizeof(O);  // column tiles turned round together: 128 bytes of a row
    constexpr int STORES = B::FM * B::FN / JO * 4;
    static_assert(B::LOADS + STORES <= 63, "the wait counter holds six bits");
    const uint32_t gm = (a.tiles + B::TA - 1) / B::TA, gn = (b.tiles + B::TB - 1) / B::TB, total = gm * gn;
    auto next = [&](Cursor& c) -> Place {
        const uint32_t l = list_place(c.first, total);
        c.first += gridDim.x;  // total and the grid are below 2^31: no wrap
        if (l >= total) return {0, 0, false};
        while (l - c.band * 8 * gn >= 8 * gn) c.band++;  // l only grows
        const uint32_t in = l - c.band * 8 * gn, rows = gm - c.band * 8 < 8 ? gm - c.band * 8 : 8, col = rows == 8 ? in / 8 : in / rows;
        return place_at((c.band * 8 + in - col * rows) * B::TA, col * B::TB);
    };
    auto finish = [&](const Place& t, f32x16 (&acc)[B::FM][B::FN]) -> bool {
        typedef O piece __attribute__((ext_vector_type(16 / sizeof(O))));
        typedef O piece_any __attribute__((ext_vector_type(16 / sizeof(O)), aligned(sizeof(O))));
        typedef O quad __attribute__((ext_vector_type(4)));
        constexpr uint32_t PE = 16 / sizeof(O);
        const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wr = wave / B::WC, wc = wave % B::WC, r = lane % 32;
        uint8_t* turn = lds + B::LDS + wave * B::OUT;
        const bool inside = (uint64_t)(t.i0 + B::TA) * 32 <= m && (uint64_t)(t.j0 + B::TB) * 32 <= n;
#pragma unroll
        for (int i = 0; i < B::FM; i++)
#pragma unroll
            for (int j0 = 0; j0 < B::FN; j0 += JO) {
#pragma unroll
                for (int j = 0; j < JO; j++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const f32x16& v = acc[i][j0 + j];
                        const quad o = {(O)(alpha * v[q * 4]), (O)(alpha * v[q * 4 + 1]), (O)(alpha * v[q * 4 + 2]), (O)(alpha * v[q * 4 + 3])};
                        const uint32_t byte = (j * 32 + q * 8 + lane / 32 * 4) * sizeof(O);
                        *reinterpret_cast<quad*>(turn + r * 128 + ((byte / 16 ^ (r & 7)) * 16 | byte % 16)) = o;
                    }
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const uint32_t rr = s * 8 + lane / 8, cc = lane % 8;
                    const piece o = *reinterpret_cast<const piece*>(turn + rr * 128 + (cc ^ (rr & 7)) * 16);
                    const uint64_t row = (uint64_t)(t.i0 + wr * B::FM + i) * 32 + rr, col = (uint64_t)(t.j0 + wc * B::FN + j0) * 32 + cc * PE;
                    O* to = c + row * cs + col;
                    if (inside) {
                        *reinterpret_cast<piece_any*>(to) = o;
                    } else if (row < m && col < n) {
                        if (n - col >= PE) {
                            *reinterpret_cast<piece_any*>(to) = o;
                        } else {
#pragma unroll
                            for (uint32_t k = 0; k < PE; k++)
                                if (col + k < n) to[k] = o[k];
                        }
                    }
                }
            }
        return inside;
    };
    mx_stream<B, STORES>(a, b, col_tiles, lds, next, [](const Place&) {}, finish);
}

// ------------------------------------------------------------------------------------------------ near pairs
// Length of every row of 4-bit values, and the least of every row tile: the root of the row's product with itself, summed by the
// same instructions in the same order as the products that it is compared with, so that equal rows have a cosine of 1 up to three
// roundings whatever their width.  (A sum in another order is off by up to 2^-15 of it at 32768 columns whose blocks differ much.)
// A wave multiplies a row tile by itself and keeps the diagonal, which of a row r is in lane r or r + 32.  A row of zeros, one
// with a NaN and one of a length outside [2^-60, 2^60], where the product of two lengths could leave the 32-bit numbers, gets
// an infinite length, which no product reaches.
__global__ __launch_bounds__(256) void mx_length_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t col_tiles,
                                                        uint64_t row_tiles, float* __restrict__ length, float* __restrict__ least,
                                                        unsigned long long* n_edges) {
    const uint32_t lane = lane_id(), r = lane % 32;
    if (blockIdx.x == 0 && threadIdx.x == 0) *n_edges = 0;
    for (uint64_t rt = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64; rt < row_tiles; rt += (uint64_t)gridDim.x * 4) {
        const uint8_t *p = codes + rt * col_tiles * TILE + lane * 16, *q = scales + rt * col_tiles * STILE + lane * 2;
        f32x16 acc = 0.0f;
#pragma unroll 4
        for (uint32_t ct = 0; ct < col_tiles; ct++) {
            const i32x4 a0 = *reinterpret_cast<const i32x4*>(p + (uint64_t)ct * TILE), a1 = *reinterpret_cast<const i32x4*>(p + (uint64_t)ct * TILE + 1024);
            const int sc = *reinterpret_cast<const uint16_t*>(q + (uint64_t)ct * STILE);
            acc = mma(a0, sc, a0, sc, acc, 0);
            acc = mma(a1, sc, a1, sc, acc, 1);
        }
        float s = 0;
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) s = i / 4 * 8 + lane / 32 * 4 + i % 4 == r ? acc[i] : s;
        const float other = __shfl_xor(s, 32, 64);
        s = r / 4 % 2 == lane / 32 ? s : other;
        s = s >= 0x1p-120f && s <= 0x1p120f ? sqrtf(s) : __builtin_inff();
        if (lane < 32) length[rt * 32 + lane] = s;
#pragma unroll
        for (int d = 16; d; d >>= 1) s = fminf(s, __shfl_xor(s, d, 64));
        if (lane == 0) least[rt] = s;
    }
}

// The product of a matrix with itself, lower triangle only; C (n^2 numbers) is never written.  A wave first compares the largest
// element of each 32 x 32 piece with min_cosine times the least lengths of its rows and columns, half an instruction per
// element; where that is reached (near pairs are rare, and so is it unless lengths differ much inside a row tile) each
// element is compared with its own two lengths, and the pairs are appended with one atomic per element position and wave.
// 45000 x 768: 395 us = 3.9 PFLOP/s of the triangle; a tile's end is a sixth of that.
template <typename B>
__global__ __launch_bounds__(B::WAVES * 64) void mx_pairs_kernel(const Packed a, uint64_t n, uint32_t col_tiles, const float* __restrict__ length,
                                                                 const float* __restrict__ least, float min_cosine, uint32_t* __restrict__ eu,
                                                                 uint32_t* __restrict__ ev, uint64_t cap, unsigned long long* __restrict__ n_edges) {
    static_assert(B::TA == B::TB, "square blocks: the diagonal ones hold both sides");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint32_t g = (a.tiles + B::TA - 1) / B::TA, bands = (g + 7) / 8, total = 32 * bands * (bands + 1);
    auto next = [&](Cursor& c) -> Place {
        for (;;) {
            const uint32_t l = list_place(c.first, total);
            c.first += gridDim.x;
            if (l >= total) return {0, 0, false};
            // band: eight block rows, 8 (band + 1) block columns, after 32 band (band + 1) places; l only grows
            while (32 * (c.band + 1) * (c.band + 2) <= l) c.band++;
            const uint32_t in = l - 32 * c.band * (c.band + 1), bi = c.band * 8 + in % 8, bj = in / 8;
            if (bi < g && bj <= bi) return place_at(bi * B::TA, bj * B::TB);
        }
    };
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wr = wave / B::WC, wc = wave % B::WC, last = a.tiles - 1;
    float li[B::FM], lj[B::FN];  // least lengths of the wave's row tiles: scalar loads, for which the tile's first step waits
    auto begin = [&](const Place& t) {
        const uint32_t it = t.i0 + wr * B::FM, jt = t.j0 + wc * B::FN;
#pragma unroll
        for (int i = 0; i < B::FM; i++) li[i] = least[it + i <= last ? it + i : last];
#pragma unroll
        for (int j = 0; j < B::FN; j++) lj[j] = least[jt + j <= last ? jt + j : last];
    };
    auto finish = [&](const Place& t, f32x16 (&acc)[B::FM][B::FN]) -> bool {
        const uint32_t lane = lane_id(), it = t.i0 + wr * B::FM, jt = t.j0 + wc * B::FN;
#pragma unroll
        for (int i = 0; i < B::FM; i++) {
            if (it + i > last) break;
#pragma unroll
            for (int j = 0; j < B::FN; j++) {
                if (jt + j > last) break;
                float top = acc[i][j][0];
#pragma unroll
                for (int k = 1; k < 16; k++) top = fmaxf(top, acc[i][j][k]);
                if (__ballot(top >= min_cosine * li[i] * lj[j]) == 0) continue;
                const uint64_t u = ((uint64_t)it + i) * 32 + lane % 32;
                const float need = u < n ? min_cosine * length[u] : __builtin_inff();
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint64_t v0 = ((uint64_t)jt + j) * 32 + q * 8 + lane / 32 * 4;
                    const f32x4 len = *reinterpret_cast<const f32x4*>(length + v0);  // filled up to whole tiles
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint64_t v = v0 + k;
                        // (an infinite length is out of reach, whatever the sum overflowed to)
                        const bool hit = acc[i][j][q * 4 + k] >= need * len[k] && need * len[k] < __builtin_inff() && v < u && u < n;
                        const uint64_t hits = __ballot(hit);
                        if (!hits) continue;
                        const int leader = __ffsll((unsigned long long)hits) - 1;
                        unsigned long long at = 0;
                        if ((int)lane == leader) at = atomicAdd(n_edges, (unsigned long long)__popcll(hits));
                        at = __shfl(at, leader, 64) + below(hits);
                        if (hit && at < cap) {
                            eu[at] = (uint32_t)u;
                            ev[at] = (uint32_t)v;
                        }
                    }
                }
            }
        }
        return false;
    };
    mx_stream<B, 0>(a, a, col_tiles, lds, next, begin, finish);
}

int check_packed(const char* who, const char* what, const void* codes, const void* scales) {
    REQUIRE(codes && scales, "%s: %s is NULL", who, what);
    REQUIRE(aligned_to(codes, 16) && aligned_to(scales, 16), "%s: codes and scales of %s must be 16-byte aligned", who, what);
    return MDD_OK;
}
template <typename K>
hipError_t allow_lds(K kernel, uint32_t bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

}  // namespace

extern "C" {

int mdd_mx_quantize(mdd_ctx* ctx, const void* x, int type, uint64_t x_stride, uint64_t n_rows, uint32_t dim, uint8_t* codes,
                    uint8_t* scales) {
    const char* who = "mdd_mx_quantize";
    REQUIRE(ctx, "%s: ctx is NULL", who);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(type_bytes(type), "%s: unknown element type %d", who, type);
    REQUIRE(n_rows <= MDD_MX_MAX_ROWS, "%s: more than 2^31 - 256 rows", who);
    if (n_rows == 0) return MDD_OK;
    REQUIRE(x && aligned_to(x, type_bytes(type)), "%s: x is NULL or not aligned to its elements", who);
    REQUIRE(x_stride >= dim, "%s: row stride %llu below dim %u", who, (unsigned long long)x_stride, dim);
    const int rc = check_packed(who, "the output", codes, scales);
    if (rc) return rc;
    ON_DEVICE(ctx);
    const uint32_t col_tiles = (dim + 127) / 128;
    const uint64_t halves = (n_rows + 31) / 32 * 2 * col_tiles, want = (halves + 3) / 4;
    const dim3 grid((unsigned)(want < (1u << 22) ? want : (1u << 22)));
    MDD_FOR_TYPE(type, T, {
        hipLaunchKernelGGL((mx_quantize_kernel<T>), grid, dim3(256), 0, ctx->stream, (const T*)x, x_stride, n_rows, dim, halves, col_tiles, codes, scales);
    });
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

int mdd_mx_matmul(mdd_ctx* ctx, const uint8_t* a_codes, const uint8_t* a_scales, uint64_t m, const uint8_t* b_codes,
                  const uint8_t* b_scales, uint64_t n, uint32_t dim, float alpha, void* c, int c_type, uint64_t c_stride) {
    const char* who = "mdd_mx_matmul";
    REQUIRE(ctx, "%s: ctx is NULL", who);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(c_type == MDD_F32 || c_type == MDD_BF16, "%s: c_type %d is neither MDD_F32 nor MDD_BF16", who, c_type);
    REQUIRE(m <= MDD_MX_MAX_ROWS && n <= MDD_MX_MAX_ROWS, "%s: more than 2^31 - 256 rows", who);
    if (m == 0 || n == 0) return MDD_OK;
    int rc = check_packed(who, "A", a_codes, a_scales);
    if (!rc) rc = check_packed(who, "B", b_codes, b_scales);
    if (rc) return rc;
    REQUIRE(c && aligned_to(c, type_bytes(c_type)), "%s: c is NULL or not aligned to its elements", who);
    REQUIRE(c_stride >= n, "%s: c_stride below n", who);
    const uint64_t at = (m + 31) / 32, bt = (n + 31) / 32;
    REQUIRE((at / Tiles::TA + 1) * (bt / Tiles::TB + 1) < MAX_TILES, "%s: m x n is above 2^31 tiles of 256 x 256", who);
    ON_DEVICE(ctx);
    const uint32_t ct = (dim + 127) / 128;
    auto run = [&](auto* out) -> hipError_t {
        typedef std::remove_pointer_t<decltype(out)> O;
        const uint64_t cus = (uint64_t)ctx->cus, groups = (at + 3) / 4;
        auto skinny = [&](const uint8_t* few_codes, const uint8_t* few_scales, uint64_t few_rows, const uint8_t* codes, const uint8_t* scales, uint64_t rows,
                          bool swapped) -> hipError_t {
            const uint64_t few = (few_rows + 31) / 32, tiles = (rows + 31) / 32;
            // one wave a row tile fills the chip from 8 waves a CU on; below that four waves share a tile's columns
            const bool split = tiles < cus * 8 && ct > 1;
            auto kernel = split ? (few == 1 ? mx_skinny_kernel<O, 1, 4> : few == 2 ? mx_skinny_kernel<O, 2, 4> : mx_skinny_kernel<O, 4, 4>)
                                : (few == 1 ? mx_skinny_kernel<O, 1, 1> : few == 2 ? mx_skinny_kernel<O, 2, 1> : mx_skinny_kernel<O, 4, 1>);
            hipLaunchKernelGGL(kernel, dim3((unsigned)(split ? tiles : (tiles + 3) / 4), (unsigned)(few <= 2 ? 1 : (few + 3) / 4)), dim3(256), 0, ctx->stream,
                               few_codes, few_scales, few_rows, (uint32_t)few, codes, scales, rows, tiles, ct, alpha, out, c_stride, swapped);
            return hipGetLastError();
        };
        // Up to 64 rows are quicker beside streamed rows of the other matrix than in tiles that stay mostly empty (64 x 262144
        // x 1024: 39 us, tiles 48; 262144 x 1 x 1024 25 and 52), and so are results too small for tiles to fill the chip, up to
        // a block a CU (1024 x 1000 x 4096: 12 us, tiles 34; with two blocks a CU both take 34).
        if (at <= 2 || bt * groups <= cus) return skinny(a_codes, a_scales, m, b_codes, b_scales, n, false);
        if (bt <= 2) return skinny(b_codes, b_scales, n, a_codes, a_scales, m, true);
        const Packed pa = {a_codes, a_scales, (uint32_t)at}, pb = {b_codes, b_scales, (uint32_t)bt};
        const uint64_t tiles = ((at + Tiles::TA - 1) / Tiles::TA) * ((bt + Tiles::TB - 1) / Tiles::TB);
        constexpr uint32_t bytes = Tiles::LDS + Tiles::WAVES * Tiles::OUT;
        const hipError_t e = allow_lds(mx_matmul_kernel<O, Tiles>, bytes);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL((mx_matmul_kernel<O, Tiles>), dim3((unsigned)(tiles < cus ? tiles : cus)), dim3(Tiles::WAVES * 64), bytes, ctx->stream, pa, m, pb,
                           n, ct, alpha, out, c_stride);
        return hipGetLastError();
    };
    HIP_TRY(c_type == MDD_F32 ? run((float*)c) : run((__bf16*)c));
    return MDD_OK;
}

uint64_t mdd_mx_pairs_ws_bytes(uint64_t m) { return round_up(round_up(m, 32) * 4, 256) + round_up((m + 31) / 32 * 4, 256); }

int mdd_mx_pairs(mdd_ctx* ctx, const uint8_t* codes, const uint8_t* scales, uint64_t m, uint32_t dim, float min_cosine,
                 uint32_t* edge_u, uint32_t* edge_v, uint64_t edge_cap, uint64_t* n_edges, void* ws, uint64_t ws_bytes) {
    const char* who = "mdd_mx_pairs";
    REQUIRE(ctx && n_edges, "%s: NULL argument", who);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(min_cosine > 0.0f && min_cosine <= 1.0f, "%s: min_cosine=%g outside (0,1]", who, (double)min_cosine);
    REQUIRE(m <= MDD_MX_MAX_PAIR_ROWS, "%s: more than 2^22 rows", who);
    REQUIRE(edge_cap == 0 || (edge_u && edge_v), "%s: NULL buffer", who);
    const uint64_t need = mdd_mx_pairs_ws_bytes(m);
    if (m) {
        const int rc = check_packed(who, "the matrix", codes, scales);
        if (rc) return rc;
        REQUIRE(ws && aligned_to(ws, 256) && ws_bytes >= need, "%s: workspace of %llu bytes, 256-byte aligned, needed", who, (unsigned long long)need);
    }
    ON_DEVICE(ctx);
    const uint64_t rt = (m + 31) / 32;
    const uint32_t ct = (dim + 127) / 128;
    auto* count = reinterpret_cast<unsigned long long*>(n_edges);
    float *length = (float*)ws, *least = length + round_up(m, 64);
    const uint64_t blocks = (rt + 3) / 4;
    hipLaunchKernelGGL(mx_length_kernel, dim3((unsigned)(blocks < 1 ? 1 : blocks)), dim3(256), 0, ctx->stream, codes, scales, ct, rt,
                       length, least, count);
    if (m) {
        const uint64_t cus = (uint64_t)ctx->cus, bands = (rt + 8 * Tiles::TA - 1) / (8 * Tiles::TA), places = 32 * bands * (bands + 1);
        HIP_TRY(allow_lds(mx_pairs_kernel<Tiles>, Tiles::LDS));
        hipLaunchKernelGGL((mx_pairs_kernel<Tiles>), dim3((unsigned)(places < cus ? places : cus)), dim3(Tiles::WAVES * 64), Tiles::LDS, ctx->stream,
                           Packed{codes, scales, (uint32_t)rt}, m, ct, length, least, min_cosine, edge_u, edge_v, edge_cap, count);
    }
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

}  // extern "C"
