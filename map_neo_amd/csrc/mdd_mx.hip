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
// code of |a| on the grid 0 .5 1 1.5 2 3 4 6: below 1 the grid is even (steps of .5); from 1 on it is a float with one
// fraction bit, so rounding the bits to that place (ties to even) and rebasing the exponent gives the code
__device__ __forceinline__ uint32_t e2m1(float a) {
    const uint32_t u = __float_as_uint(a);
    const uint32_t hi = ((u + 0x1FFFFFu + (u >> 22 & 1u)) >> 22) - 252u;
    return a < 1.0f ? (uint32_t)rintf(a + a) : (hi < 7u ? hi : 7u);
}

// A thread takes a block of 32 columns of a row; four threads side by side take a tile's four blocks, 32 rows a tile.
// Bound by HBM: the matrix is read once, a bit more than half a byte per element is written.
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, uint64_t stride, uint64_t n_rows, uint32_t dim,
                                                          uint64_t n_tiles, uint32_t col_tiles, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
    const uint32_t t = threadIdx.x % 128, kb = t % 4, r = t / 4;
    for (uint64_t tile = (uint64_t)blockIdx.x * 2 + threadIdx.x / 128; tile < n_tiles; tile += (uint64_t)gridDim.x * 2) {
        const uint64_t rt = tile / col_tiles, row = rt * 32 + r;
        const uint32_t ct = (uint32_t)(tile - rt * col_tiles), col = ct * 128 + kb * 32;
        f32x8 v[4];
        uint32_t big = 0;
        const bool in = row < n_rows && col < dim;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            v[c] = 0.0f;
            if (in && col + c * 8 < dim) v[c] = load8<T>(x + row * stride + col + c * 8, dim - col - c * 8);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint32_t m = __float_as_uint(v[c][k]) & 0x7FFFFFFFu;
                big = m > big ? m : big;
            }
        }
        // biased exponent of the largest, less 2; subnormal and zero blocks stop at 2^-127
        const int e = (int)(big >> 23) - 127 - 2, sc = e > -127 ? e : -127;
        const bool bad = big >= 0x7F800000u;
        const float inv = __uint_as_float((uint32_t)(127 - sc) << 23);  // sc is -127 .. 125: 2^2 .. 2^254 of the exponent field
        u32x4 p = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint32_t w = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint32_t sign = __float_as_uint(v[c][k]) >> 31;
                w |= (e2m1(fabsf(v[c][k]) * inv) | sign << 3) << (4 * k);
            }
            p[c] = bad ? 0u : w;
        }
        *reinterpret_cast<u32x4*>(codes + tile * TILE + kb * 512 + r * 16) = p;
        scales[tile * STILE + (kb & 1) * 64 + r * 2 + (kb >> 1)] = (uint8_t)(!in ? 127 : bad ? 255 : sc + 127);
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

// Few rows of A (FM row tiles): every wave streams one row tile of B from memory, the A fragments come out of the caches.
// Bound by reading B.  SPLIT waves share a tile's columns where there are too few tiles to fill the chip; their sums are
// joined in LDS in wave order.
template <typename O, int FM, int SPLIT>
__global__ __launch_bounds__(256) void mx_skinny_kernel(const uint8_t* __restrict__ ac, const uint8_t* __restrict__ as, uint64_t m, uint32_t a_tiles,
                                                        const uint8_t* __restrict__ bc, const uint8_t* __restrict__ bs, uint64_t n, uint64_t b_tiles,
                                                        uint32_t col_tiles, float alpha, O* __restrict__ c, uint64_t cs) {
    constexpr int U = FM == 1 ? 4 : 2;  // column tiles in flight
    __shared__ float join[SPLIT > 1 ? (SPLIT - 1) * FM * 16 * 64 : 1];
    const uint32_t lane = lane_id(), wave = threadIdx.x / 64, part = wave % SPLIT;
    const uint64_t tile = (uint64_t)blockIdx.x * (4 / SPLIT) + wave / SPLIT;
    f32x16 acc[FM];
#pragma unroll
    for (int f = 0; f < FM; f++) acc[f] = 0.0f;
    if (tile < b_tiles) {
        const uint8_t *bp = bc + tile * col_tiles * TILE + lane * 16, *sp = bs + tile * col_tiles * STILE + lane * 2;
        const uint8_t *ap = ac + lane * 16, *tp = as + lane * 2;
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
                    const uint64_t at = (uint64_t)(f < (int)a_tiles ? f : a_tiles - 1) * col_tiles + k;
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
        const uint64_t row = f * 32 + lane % 32;
        if (row >= m) continue;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint64_t col = tile * 32 + q * 8 + lane / 32 * 4;
            if (col < n)
                store_quad<O>(c + row * cs + col, (uint32_t)(n - col < 4 ? n - col : 4), alpha * acc[f][q * 4], alpha * acc[f][q * 4 + 1],
                              alpha * acc[f][q * 4 + 2], alpha * acc[f][q * 4 + 3]);
        }
    }
}

// Tiled product.  A block of WR x WC waves computes (WR * FM * 32) x (WC * FN * 32) of C.  Column tiles (128 columns) go from
// memory straight into LDS, three in rotation: while one is multiplied, the next is complete or landing and the one after is
// requested, so a load has two steps to arrive and a step needs one barrier (behind it every wave is done with the buffer
// that is requested next).
template <int WR, int WC, int FM, int FN>
struct Block {
    static constexpr int WAVES = WR * WC, TA = WR * FM, TB = WC * FN, TILES = TA + TB, PER_WAVE = TILES / WAVES;
    static constexpr uint32_t STAGE = TILES * (TILE + STILE), LDS = 3 * STAGE;
    static constexpr int LOADS = PER_WAVE * 2 + 1;  // per wave and step: two halves of each of its tiles, and their scales
    static_assert(TILES % WAVES == 0 && PER_WAVE * 8 <= 64, "every wave loads whole tiles, their scales in one instruction");
};

__device__ __forceinline__ void to_lds(const uint8_t* g, uint8_t* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)g, (__attribute__((address_space(3))) uint32_t*)l, 16, 0, 0);
}

template <int WR, int WC, int FM, int FN>
__device__ __forceinline__ void mx_tile(const uint8_t* __restrict__ ac, const uint8_t* __restrict__ as, uint64_t a0, uint64_t a_tiles,
                                        const uint8_t* __restrict__ bc, const uint8_t* __restrict__ bs, uint64_t b0, uint64_t b_tiles,
                                        uint32_t col_tiles, uint8_t* lds, f32x16 (&acc)[FM][FN]) {
    using B = Block<WR, WC, FM, FN>;
    const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wr = wave / WC, wc = wave % WC;
    // this wave's share of a step's loads: PER_WAVE tiles; row tiles past the end repeat the last one (their results are not used)
    const uint8_t* src[B::PER_WAVE];
#pragma unroll
    for (int i = 0; i < B::PER_WAVE; i++) {
        const uint32_t t = wave * B::PER_WAVE + i;
        const bool is_a = t < B::TA;
        uint64_t rt = is_a ? a0 + t : b0 + t - B::TA;
        const uint64_t last = (is_a ? a_tiles : b_tiles) - 1;
        rt = rt < last ? rt : last;
        src[i] = (is_a ? ac : bc) + rt * col_tiles * TILE + lane * 16;
    }
    const uint8_t* ssrc;
    {
        const uint32_t t = wave * B::PER_WAVE + (lane / 8 < B::PER_WAVE ? lane / 8 : 0);
        const bool is_a = t < B::TA;
        uint64_t rt = is_a ? a0 + t : b0 + t - B::TA;
        const uint64_t last = (is_a ? a_tiles : b_tiles) - 1;
        rt = rt < last ? rt : last;
        ssrc = (is_a ? as : bs) + rt * col_tiles * STILE + lane % 8 * 16;
    }
    auto request = [&](uint32_t k, uint32_t buf) {
        uint8_t* to = lds + buf * B::STAGE;
#pragma unroll
        for (int i = 0; i < B::PER_WAVE; i++) {
            uint8_t* l = to + (wave * B::PER_WAVE + i) * TILE;
            to_lds(src[i] + (uint64_t)k * TILE, l);
            to_lds(src[i] + (uint64_t)k * TILE + 1024, l + 1024);
        }
        if (lane < B::PER_WAVE * 8) to_lds(ssrc + (uint64_t)k * STILE, to + B::TILES * TILE + wave * B::PER_WAVE * STILE);
    };
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = 0.0f;
    request(0, 0);
    if (col_tiles > 1) request(1, 1);
    uint32_t buf = 0;
#pragma unroll 1
    for (uint32_t k = 0; k < col_tiles; k++) {
        // the loads of step k are in LDS once at most those of step k + 1 are outstanding; and this wave has read all that
        // it wants of the buffer of step k - 1, which is requested anew behind the barrier
        if (k + 1 < col_tiles) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(B::LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (k + 2 < col_tiles) request(k + 2, buf == 0 ? 2 : buf - 1);
        const uint8_t *la = lds + buf * B::STAGE + (wr * FM) * TILE, *lb = lds + buf * B::STAGE + (B::TA + wc * FN) * TILE;
        const uint8_t *sa = lds + buf * B::STAGE + B::TILES * TILE + (wr * FM) * STILE, *sb = lds + buf * B::STAGE + B::TILES * TILE + (B::TA + wc * FN) * STILE;
        int xa[FM], xb[FN];
#pragma unroll
        for (int i = 0; i < FM; i++) xa[i] = *reinterpret_cast<const uint16_t*>(sa + i * STILE + lane * 2);
#pragma unroll
        for (int j = 0; j < FN; j++) xb[j] = *reinterpret_cast<const uint16_t*>(sb + j * STILE + lane * 2);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            i32x4 a[FM], b[FN];
#pragma unroll
            for (int i = 0; i < FM; i++) a[i] = *reinterpret_cast<const i32x4*>(la + i * TILE + h * 1024 + lane * 16);
#pragma unroll
            for (int j = 0; j < FN; j++) b[j] = *reinterpret_cast<const i32x4*>(lb + j * TILE + h * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = mma(b[j], xb[j], a[i], xa[i], acc[i][j], h);
        }
        buf = buf == 2 ? 0 : buf + 1;
    }
    __syncthreads();  // the next tile's first loads go into buffers that a slower wave may still be reading
}

// Work order.  Blocks go to the eight XCDs in turn, so XCD x gets a run of consecutive tiles of the list, and the list walks
// eight row tiles at a time down the columns: the 32 blocks that an XCD runs together share 8 + 4 tiles out of its L2.
__device__ __forceinline__ uint64_t xcd_order(uint64_t b, uint64_t n) {
    const uint64_t per = n / 8;  // the last n % 8 keep their place
    return b < per * 8 ? (b % 8) * per + b / 8 : b;
}

template <typename O, int WR, int WC, int FM, int FN>
__global__ __launch_bounds__(WR * WC * 64) void mx_matmul_kernel(const uint8_t* __restrict__ ac, const uint8_t* __restrict__ as, uint64_t m, uint64_t a_tiles,
                                                                 const uint8_t* __restrict__ bc, const uint8_t* __restrict__ bs, uint64_t n,
                                                                 uint64_t b_tiles, uint32_t col_tiles, float alpha, O* __restrict__ c, uint64_t cs) {
    using B = Block<WR, WC, FM, FN>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint64_t gm = (a_tiles + B::TA - 1) / B::TA, gn = (b_tiles + B::TB - 1) / B::TB, total = gm * gn;
    for (uint64_t t = blockIdx.x; t < total; t += gridDim.x) {
        const uint64_t first = t - blockIdx.x, here = total - first < gridDim.x ? total - first : gridDim.x;
        const uint64_t l = first + xcd_order(blockIdx.x, here);
        const uint64_t band = l / (8 * gn), rows = gm - band * 8 < 8 ? gm - band * 8 : 8, in = l - band * 8 * gn;
        const uint64_t i0 = (band * 8 + in % rows) * B::TA, j0 = in / rows * B::TB;
        f32x16 acc[FM][FN];
        mx_tile<WR, WC, FM, FN>(ac, as, i0, a_tiles, bc, bs, j0, b_tiles, col_tiles, lds, acc);
        const uint32_t lane = lane_id(), wave = threadIdx.x / 64, wr = wave / WC, wc = wave % WC;
#pragma unroll
        for (int i = 0; i < FM; i++) {
            const uint64_t row = (i0 + wr * FM + i) * 32 + lane % 32;
            if (row >= m) continue;
#pragma unroll
            for (int j = 0; j < FN; j++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint64_t col = (j0 + wc * FN + j) * 32 + q * 8 + lane / 32 * 4;
                    if (col < n)
                        store_quad<O>(c + row * cs + col, (uint32_t)(n - col < 4 ? n - col : 4), alpha * acc[i][j][q * 4], alpha * acc[i][j][q * 4 + 1],
                                      alpha * acc[i][j][q * 4 + 2], alpha * acc[i][j][q * 4 + 3]);
                }
        }
    }
}

// ------------------------------------------------------------------------------------------------ near pairs
// Length of every row of 4-bit values.  The magnitudes (doubled: 0 1 2 3 4 6 8 12) are looked up four at a time with a byte
// permute and squared with a byte dot product: a block of 32 columns is summed in whole numbers.  A row of zeros gets an
// infinite length, which no product reaches.
__global__ __launch_bounds__(128) void mx_length_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t col_tiles,
                                                        uint64_t row_tiles, float* __restrict__ length, unsigned long long* n_edges) {
    __shared__ float lds[4][32];
    const uint32_t kb = threadIdx.x / 32, r = threadIdx.x % 32;
    if (blockIdx.x == 0 && threadIdx.x == 0) *n_edges = 0;
    for (uint64_t rt = blockIdx.x; rt < row_tiles; rt += gridDim.x) {
        float s = 0;
        for (uint32_t ct = 0; ct < col_tiles; ct++) {
            const uint64_t tile = rt * col_tiles + ct;
            const u32x4 p = *reinterpret_cast<const u32x4*>(codes + tile * TILE + kb * 512 + r * 16);
            const int e = (int)scales[tile * STILE + (kb & 1) * 64 + r * 2 + (kb >> 1)];
            int sq = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t lo = __builtin_amdgcn_perm(0x0C080604u, 0x03020100u, p[k] & 0x07070707u);
                const uint32_t hi = __builtin_amdgcn_perm(0x0C080604u, 0x03020100u, p[k] >> 4 & 0x07070707u);
                sq = __builtin_amdgcn_sdot4((int)lo, (int)lo, sq, false);
                sq = __builtin_amdgcn_sdot4((int)hi, (int)hi, sq, false);
            }
            s += e == 255 ? __builtin_nanf("") : ldexpf((float)sq, 2 * (e - 127) - 2);
        }
        lds[kb][r] = s;
        __syncthreads();
        if (kb == 0) {
            s = lds[0][r] + lds[1][r] + lds[2][r] + lds[3][r];
            length[rt * 32 + r] = s == 0.0f ? __builtin_inff() : sqrtf(s);
        }
        __syncthreads();
    }
}

// The product of a matrix with itself, lower triangle only; instead of storing C a lane compares each element with
// min_cosine times the two lengths and appends the pairs that reach it.  Pairs are rare, so the append may cost: one atomic
// per element position and wave that holds any.  C (n^2 numbers) is never written.
template <int WR, int WC, int FM, int FN>
__global__ __launch_bounds__(WR * WC * 64) void mx_pairs_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint64_t n,
                                                                uint64_t row_tiles, uint32_t col_tiles, const float* __restrict__ length, float min_cosine,
                                                                uint32_t* __restrict__ eu, uint32_t* __restrict__ ev, uint64_t cap,
                                                                unsigned long long* __restrict__ n_edges) {
    using B = Block<WR, WC, FM, FN>;
    static_assert(B::TA == B::TB, "square blocks: the diagonal ones hold both sides");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint64_t g = (row_tiles + B::TA - 1) / B::TA, bands = (g + 7) / 8, total = 32 * bands * (bands + 1);
    for (uint64_t t = blockIdx.x; t < total; t += gridDim.x) {
        const uint64_t first = t - blockIdx.x, here = total - first < gridDim.x ? total - first : gridDim.x;
        const uint64_t l = first + xcd_order(blockIdx.x, here);
        // band b: eight block rows, 8 (b + 1) block columns, after 32 b (b + 1) places
        uint64_t b = (uint64_t)((__builtin_sqrtf(1.0f + (float)l / 8.0f) - 1.0f) * 0.5f);
        while (32 * b * (b + 1) > l) b--;
        while (32 * (b + 1) * (b + 2) <= l) b++;
        const uint64_t in = l - 32 * b * (b + 1), bi = b * 8 + in % 8, bj = in / 8;
        if (bi >= g || bj > bi) continue;  // the same for the whole block
        const uint64_t i0 = bi * B::TA, j0 = bj * B::TB;
        f32x16 acc[FM][FN];
        mx_tile<WR, WC, FM, FN>(codes, scales, i0, row_tiles, codes, scales, j0, row_tiles, col_tiles, lds, acc);
        const uint32_t lane = lane_id(), wave = threadIdx.x / 64, wr = wave / WC, wc = wave % WC;
#pragma unroll
        for (int i = 0; i < FM; i++) {
            const uint64_t u = (i0 + wr * FM + i) * 32 + lane % 32;
            const float need = u < n ? min_cosine * length[u] : __builtin_inff();
#pragma unroll
            for (int j = 0; j < FN; j++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint64_t v0 = (j0 + wc * FN + j) * 32 + q * 8 + lane / 32 * 4;
                    f32x4 len = __builtin_inff();
                    if (v0 < row_tiles * 32) len = *reinterpret_cast<const f32x4*>(length + v0);  // filled up to whole tiles
                    bool any = false;
#pragma unroll
                    for (int k = 0; k < 4; k++) any |= acc[i][j][q * 4 + k] >= need * len[k];
                    if (__ballot(any) == 0) continue;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint64_t v = v0 + k;
                        // (an infinite product of lengths is out of reach, whatever the sum overflowed to)
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
}

using Big = Block<2, 4, 4, 2>;    // 256 x 256, 8 waves
using Small = Block<2, 2, 2, 2>;  // 128 x 128, 4 waves

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
    REQUIRE(n_rows < (1ull << 31), "%s: 2^31 or more rows", who);
    if (n_rows == 0) return MDD_OK;
    REQUIRE(x && aligned_to(x, type_bytes(type)), "%s: x is NULL or not aligned to its elements", who);
    REQUIRE(x_stride >= dim, "%s: row stride %llu below dim %u", who, (unsigned long long)x_stride, dim);
    const int rc = check_packed(who, "the output", codes, scales);
    if (rc) return rc;
    ON_DEVICE(ctx);
    const uint32_t col_tiles = (dim + 127) / 128;
    const uint64_t tiles = (n_rows + 31) / 32 * col_tiles, want = (tiles + 1) / 2;
    const dim3 grid((unsigned)(want < (1u << 22) ? want : (1u << 22)));
    MDD_FOR_TYPE(type, T, {
        hipLaunchKernelGGL((mx_quantize_kernel<T>), grid, dim3(256), 0, ctx->stream, (const T*)x, x_stride, n_rows, dim, tiles, col_tiles, codes, scales);
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
    REQUIRE(m < (1ull << 31) && n < (1ull << 31), "%s: 2^31 or more rows", who);
    if (m == 0 || n == 0) return MDD_OK;
    int rc = check_packed(who, "A", a_codes, a_scales);
    if (!rc) rc = check_packed(who, "B", b_codes, b_scales);
    if (rc) return rc;
    REQUIRE(c && aligned_to(c, type_bytes(c_type)), "%s: c is NULL or not aligned to its elements", who);
    REQUIRE(c_stride >= n, "%s: c_stride below n", who);
    ON_DEVICE(ctx);
    const uint64_t at = (m + 31) / 32, bt = (n + 31) / 32;
    const uint32_t ct = (dim + 127) / 128;
    auto run = [&](auto* out) -> hipError_t {
        typedef std::remove_pointer_t<decltype(out)> O;
        if (at <= 4) {
            // one wave a row tile of B fills the chip from 8 waves a CU on; below that four waves share a tile's columns
            const bool split = bt < (uint64_t)ctx->cus * 8 && ct > 1;
            auto kernel = split ? (at == 1 ? mx_skinny_kernel<O, 1, 4> : at == 2 ? mx_skinny_kernel<O, 2, 4> : mx_skinny_kernel<O, 4, 4>)
                                : (at == 1 ? mx_skinny_kernel<O, 1, 1> : at == 2 ? mx_skinny_kernel<O, 2, 1> : mx_skinny_kernel<O, 4, 1>);
            hipLaunchKernelGGL(kernel, dim3((unsigned)(split ? bt : (bt + 3) / 4)), dim3(256), 0, ctx->stream, a_codes, a_scales, m, (uint32_t)at, b_codes,
                               b_scales, n, bt, ct, alpha, out, c_stride);
            return hipGetLastError();
        }
        const uint64_t big = ((at + Big::TA - 1) / Big::TA) * ((bt + Big::TB - 1) / Big::TB), cap = 1u << 22;
        if (big >= (uint64_t)ctx->cus) {  // large blocks read a quarter less from L2 per product; smaller ones where they would leave CUs idle
            auto kernel = mx_matmul_kernel<O, 2, 4, 4, 2>;
            hipError_t e = allow_lds(kernel, Big::LDS);
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL(kernel, dim3((unsigned)(big < cap ? big : cap)), dim3(Big::WAVES * 64), Big::LDS, ctx->stream, a_codes, a_scales, m, at, b_codes,
                               b_scales, n, bt, ct, alpha, out, c_stride);
        } else {
            const uint64_t small = ((at + Small::TA - 1) / Small::TA) * ((bt + Small::TB - 1) / Small::TB);
            auto kernel = mx_matmul_kernel<O, 2, 2, 2, 2>;
            hipError_t e = allow_lds(kernel, Small::LDS);
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL(kernel, dim3((unsigned)(small < cap ? small : cap)), dim3(Small::WAVES * 64), Small::LDS, ctx->stream, a_codes, a_scales, m, at,
                               b_codes, b_scales, n, bt, ct, alpha, out, c_stride);
        }
        return hipGetLastError();
    };
    HIP_TRY(c_type == MDD_F32 ? run((float*)c) : run((__bf16*)c));
    return MDD_OK;
}

uint64_t mdd_mx_pairs_ws_bytes(uint64_t m) { return round_up(round_up(m, 32) * 4, 256); }

int mdd_mx_pairs(mdd_ctx* ctx, const uint8_t* codes, const uint8_t* scales, uint64_t m, uint32_t dim, float min_cosine,
                 uint32_t* edge_u, uint32_t* edge_v, uint64_t edge_cap, uint64_t* n_edges, void* ws, uint64_t ws_bytes) {
    const char* who = "mdd_mx_pairs";
    REQUIRE(ctx && n_edges, "%s: NULL argument", who);
    REQUIRE(dim >= 1 && dim <= MDD_VEC_MAX_DIM, "%s: dim=%u outside [1,%d]", who, dim, MDD_VEC_MAX_DIM);
    REQUIRE(min_cosine > 0.0f && min_cosine <= 1.0f, "%s: min_cosine=%g outside (0,1]", who, (double)min_cosine);
    REQUIRE(m < (1ull << 31), "%s: 2^31 or more rows", who);
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
    hipLaunchKernelGGL(mx_length_kernel, dim3((unsigned)(rt < 1 ? 1 : rt < (1u << 20) ? rt : (1u << 20))), dim3(128), 0, ctx->stream, codes, scales, ct, rt,
                       (float*)ws, count);
    if (m) {
        auto bands = [&](uint64_t t) { return ((rt + t - 1) / t + 7) / 8; };
        const uint64_t b = bands(Big::TA), big = (rt + Big::TA - 1) / Big::TA, cap = 1u << 22;
        if (big * (big + 1) / 2 >= (uint64_t)ctx->cus) {
            const uint64_t total = 32 * b * (b + 1);
            HIP_TRY(allow_lds(mx_pairs_kernel<2, 4, 4, 2>, Big::LDS));
            hipLaunchKernelGGL((mx_pairs_kernel<2, 4, 4, 2>), dim3((unsigned)(total < cap ? total : cap)), dim3(Big::WAVES * 64), Big::LDS, ctx->stream, codes,
                               scales, m, rt, ct, (const float*)ws, min_cosine, edge_u, edge_v, edge_cap, count);
        } else {
            const uint64_t s = bands(Small::TA), total = 32 * s * (s + 1);
            HIP_TRY(allow_lds(mx_pairs_kernel<2, 2, 2, 2>, Small::LDS));
            hipLaunchKernelGGL((mx_pairs_kernel<2, 2, 2, 2>), dim3((unsigned)(total < cap ? total : cap)), dim3(Small::WAVES * 64), Small::LDS, ctx->stream,
                               codes, scales, m, rt, ct, (const float*)ws, min_cosine, edge_u, edge_v, edge_cap, count);
        }
    }
    HIP_TRY(hipGetLastError());
    return MDD_OK;
}

}  // extern "C"
