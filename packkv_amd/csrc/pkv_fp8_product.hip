// Products of matrices in their 8-bit form (pkv_fp8.hip): y[m, n] = sum over blocks b of 128 of
//     sx[m, b] * sw[n / 128, b] * sum_{k in b} cx[m, k] * cw[n, k]        (+ bias[n]),
// rounded once to 16 bits, and the gated feed-forward of it: rows 0 .. I-1 of w give g, rows I .. 2I-1 give u, the result is
// g / (1 + exp(-g)) * u.
//
// One v_mfma_f32_16x16x128_f8f6f4 is one block's sum for 16 x 16 results: it starts from zero, and its four numbers a lane are
// added to the fp32 sums with the two scales, one fma each.  (The scales' product is rounded to fp32: below 2^-126 by up to 2^-150, times at
// most 128 * 448^2 in a block's sum.  Either scale by itself would cost four more instructions a product.)  Weights are the instruction's
// rows and x its columns, so a lane holds four neighbouring outputs of one row of x: its scale is one number a lane, the weights' scale one a
// wavefront.  The order of the 128 within a block does not matter, so lanes load what lies well: of each 128 the 16-byte pieces g and 4 + g,
// g = lane / 16.
//
// What the instruction loses: in each group of eight neighbouring k it cuts every product towards zero to a multiple of 2^-13 of the
// group's largest power of two, and adds groups in fp32 (measured).  Products of values with 4 significant bits, which are 2^-4 off
// themselves, come out 2^-13 of the largest of eight off at most; sums of 128 normal products 1.3e-5.  Results are 16-bit (half a step is 2^-8
// of a value in bf16, 2^-11 in fp16).
#include "pkv_fp8.hpp"
#include "pkv_runtime.hpp"

namespace pkv {

struct ProductParams {
    const uint8_t *x, *w;
    const float *x_scale, *w_scale;
    const uint16_t *bias;
    uint16_t *out;
    int64_t x_row, w_row, out_row, xs_row, xs_col, ws_row, ws_col;
    uint32_t rows, width, cols;          // of x; results a row (of w: twice as many rows where gated)
    uint32_t blocks;                     // of 128 along the width
    bool past;                           // results go past the caches
    bool whole4, whole8;                 // rows and their ends at multiples of four, of eight results, in memory too
};

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
// The weights' scales are scalar loads: nothing writes them while a kernel runs.
typedef const __attribute__((address_space(4))) float scalar_float;

__device__ __forceinline__ f32x4 block_product(i32x8 w, i32x8 x) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, zero, 0, 0, 0, 0, 0, 0);
}
constexpr uint32_t kNowhere = 0x80000000u;             // a buffer offset behind any tile: loads give zeroes
// Rows first .. first + count - 1 of a matrix of `rows` rows as a buffer: what lies behind its last row reads as zero.  (Scalars by force: the
// compiler would loop over the lanes of a descriptor that it formed in vector registers.)
__device__ __forceinline__ u32x4_t tile_words(const uint8_t *base, int64_t row, uint32_t first, uint32_t rows, uint32_t count, uint32_t width) {
    const uint32_t there = first < rows ? min(count, rows - first) : 0u;
    const uint64_t a = (uint64_t)(reinterpret_cast<uintptr_t>(base) + (uint64_t)((int64_t)first * row));
    return (u32x4_t){(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a), (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xFFFFu),
                     (uint32_t)__builtin_amdgcn_readfirstlane(there ? (there - 1u) * (uint32_t)row + width : 0u), 0x00020000u};
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(u32x4_t w) {
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>((uint64_t)w[0] | (uint64_t)w[1] << 32), 0, (int)w[2], 0x00020000);
}
// 16 bytes a lane from a buffer straight into LDS at `lds` + 16 lane (the compiler sees neither the copy nor its wait, copies_done()).  The
// s_nop: wait states between a write of a scalar operand by the compiler and its use here.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy_piece(u32x4_t rsrc, uint32_t lds, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(lds), "v"(off), "s"(rsrc) : "memory", "m0");
}
__device__ __forceinline__ void copy_word(u32x4_t rsrc, uint32_t lds, uint32_t off) {           // 4 bytes a lane, to lds + 4 lane
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds" :: "s"(lds), "v"(off), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop
// This wavefront's copies have arrived and its reads of LDS are done, and so for all wavefronts of the workgroup.
template <int N> __device__ __forceinline__ void copies_but() {            // (all but the last N of the wavefront's copies)
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// Results n .. n + 3 from the sums (of gate, y, and of up, u), rounded.  g / (1 + e^-g) goes through the hardware's exponential (its argument, times
// log2 e, is rounded: |g| 2^-23 of the result at most) and reciprocal (off by a step of fp32 at most), both far below 16 bits.  The reciprocal is that
// of a quarter of the sum, which stays a normal number up to the largest e^-g, and meets a quarter of up first: with g it would be 4 g, past fp32 from
// 2^126 on.  (A quarter of g instead: gated 4096 x 4096 x 2 x 12288 339 us, so 336.)
template <int DT, bool GATED> __device__ __forceinline__ u32x2 four_results(const ProductParams &p, uint32_t n, f32x4 y, f32x4 u) {
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        z[e] = y[e];
        if (GATED) z[e] = z[e] * (__builtin_amdgcn_rcpf(fmaf(__expf(-z[e]), .25f, .25f)) * (.25f * u[e]));
        else if (p.bias) z[e] += wide16<DT>(p.bias[min(n + e, p.cols - 1u)], 0);
    }
    return (u32x2){pair16<DT>(z[0], z[1]), pair16<DT>(z[2], z[3])};
}
__device__ __forceinline__ void store_four(const ProductParams &p, uint32_t m, uint32_t n, u32x2 v) {
    uint16_t *out = p.out + (int64_t)m * p.out_row + n;
    if (p.whole4) {                                        // rows and their ends at multiples of four results
        *reinterpret_cast<u32x2 *>(out) = v;
        return;
    }
    out[0] = (uint16_t)v[0];
    if (n + 1 < p.cols) out[1] = (uint16_t)(v[0] >> 16);
    if (n + 2 < p.cols) out[2] = (uint16_t)v[1];
    if (n + 3 < p.cols) out[3] = (uint16_t)(v[1] >> 16);
}

// Few rows of x: a workgroup has 16 RT rows of weights (of gate and of up each, where gated) and 16 MT rows of x.  Its eight wavefronts take the
// blocks of the width in turn, each through LDS of its own, the next block on its way while one is multiplied, without a barrier until they
// join their sums.  (Loaded straight into registers, neighbouring lanes are on different rows, and a load takes 64 cycles for the 16 of whole
// lines: 48 x 4096 x 6144 12.5 us, 7.9 this way.  Four wavefronts with two places each: 8.7.)  Bound by the weights' bytes, 1 x 12288 x 4096 9.4 us (5.4 TB/s),
// 1 x 4096 x 2 x 12288 gated 17.3 (5.8), and by the launch and the first blocks' way from memory where those are few.
template <int DT, int RT, int MT, bool GATED>
__global__ void __launch_bounds__(512) product_few_kernel(const ProductParams p) {
    constexpr int WAVES = 8, S = GATED ? 2 : 1, UNITS = S * RT, TILES = UNITS * MT;
    constexpr int kScales = (UNITS + MT) * 2048, kStage = kScales + 256;
    constexpr int kRing = WAVES * kStage, kPart = WAVES * TILES * 1024, kLds = kRing > kPart ? kRing : kPart;
    static_assert(MT <= 4, "64 scales of x");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r = lane & 15u, g = lane >> 4;
    // Workgroups go to the eight XCDs in turn: those that share rows of weights follow each other on one.
    const uint32_t tiles_n = (p.cols + 16u * RT - 1u) / (16u * RT), tiles_m = (p.rows + 16u * MT - 1u) / (16u * MT);
    const uint32_t at = (blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (at >= tiles_n * tiles_m) return;
    const uint32_t tile_n = __builtin_amdgcn_readfirstlane(at / tiles_m), tile_m = __builtin_amdgcn_readfirstlane(at - at / tiles_m * tiles_m);
    const uint32_t n0 = tile_n * 16u * RT, m0 = tile_m * 16u * MT;
    const uint32_t w_rows = S * p.cols;
    u32x4_t wr[S];
    scalar_float *ws[UNITS];
#pragma unroll
    for (int s = 0; s < S; s++) {
        const uint32_t first = n0 + (uint32_t)s * p.cols;
        wr[s] = tile_words(p.w, p.w_row, first, GATED && s == 0 ? p.cols : w_rows, 16u * RT, p.width);
#pragma unroll
        for (int i = 0; i < RT; i++) ws[s * RT + i] = (scalar_float *)(p.w_scale + (int64_t)(min(first + 16u * i, w_rows - 1u) / 128u) * p.ws_row);
    }
    const u32x4_t xr = tile_words(p.x, p.x_row, m0, p.rows, 16u * MT, p.width);
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(lds) + wave * kStage;
    const uint32_t piece = 16u * ((lane & 7u) ^ (lane >> 3)), w_off = (lane >> 3) * (uint32_t)p.w_row + piece, x_off = (lane >> 3) * (uint32_t)p.x_row + piece;
    const uint32_t scale_off = 4u * (min(m0 + lane, p.rows - 1u) - m0) * (uint32_t)p.xs_row, last = p.blocks - 1u;
    const uint64_t scale_base = reinterpret_cast<uintptr_t>(p.x_scale + (int64_t)m0 * p.xs_row);
    auto copy_block = [&](uint32_t b) {                    // (behind the last block zeroes, from no memory)
        const uint32_t k = 128u * b;
        const bool inside = k + piece < p.width;           // (a multiple of 16)
#pragma unroll
        for (int u = 0; u < UNITS; u++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                copy_piece(wr[u / RT], lds0 + u * 2048 + h * 1024, inside ? w_off + (16u * (u % RT) + 8u * h) * (uint32_t)p.w_row + k : kNowhere);
#pragma unroll
        for (int j = 0; j < 2 * MT; j++) copy_piece(xr, lds0 + UNITS * 2048 + j * 1024, inside ? x_off + 8u * j * (uint32_t)p.x_row + k : kNowhere);
        const uint64_t a = scale_base + 4u * (uint64_t)(min(b, last) * p.xs_col);
        copy_word((u32x4_t){(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a), (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xFFFFu), 0x7FFFFFFFu, 0x00020000u},
                  lds0 + kScales, scale_off);
    };
    f32x4 acc[UNITS][MT];
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[u][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const uint32_t read0 = r * 128u + 16u * (g ^ (r & 7u));
    float wf[UNITS];
    auto load_w_scales = [&](uint32_t b) {
#pragma unroll
        for (int u = 0; u < UNITS; u++) wf[u] = ws[u][(int64_t)min(b, last) * p.ws_col];
    };
    load_w_scales(wave);
    copy_block(wave);
    const uint8_t *q = lds + wave * kStage;
    for (uint32_t b = wave; b < p.blocks; b += WAVES) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        auto read_rows = [&](int tile) -> i32x8 {
            const u32x4_t lo = *reinterpret_cast<const u32x4_t *>(q + tile * 2048 + read0), hi = *reinterpret_cast<const u32x4_t *>(q + tile * 2048 + (read0 ^ 64u));
            return (i32x8){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
        };
        i32x8 wv[UNITS], xv[MT];
        float xf[MT], wn[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; u++) wv[u] = read_rows(u);
#pragma unroll
        for (int j = 0; j < MT; j++) {
            xv[j] = read_rows(UNITS + j);
            xf[j] = *reinterpret_cast<const float *>(q + kScales + 4 * (16 * j + (int)r));
        }
#pragma unroll
        for (int u = 0; u < UNITS; u++) wn[u] = wf[u];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // (read, before the next copies take the place)
        load_w_scales(b + WAVES);
        copy_block(b + WAVES);
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int u = 0; u < UNITS; u++) {
                const f32x4 d = block_product(wv[u], xv[j]);
                const float f = xf[j] * wn[u];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[u][j][e] = fmaf(d[e], f, acc[u][j][e]);
            }
    }
    copies_done();                                         // (none may arrive where the sums lie)
    f32x4 *part = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
        for (int j = 0; j < MT; j++) part[(wave * TILES + u * MT + j) * 64 + lane] = acc[u][j];
    __syncthreads();
    for (uint32_t t = wave; t < (uint32_t)(RT * MT); t += WAVES) {
        f32x4 y[S];
#pragma unroll
        for (int s = 0; s < S; s++) {
            y[s] = part[(s * RT * MT + t) * 64 + lane];
#pragma unroll
            for (int v = 1; v < WAVES; v++)
#pragma unroll
                for (int e = 0; e < 4; e++) y[s][e] += part[(v * TILES + s * RT * MT + t) * 64 + lane][e];
        }
        const uint32_t m = m0 + 16u * (t % MT) + r, n = n0 + 16u * (t / MT) + 4u * g;
        if (m < p.rows && n < p.cols) store_four(p, m, n, four_results<DT, GATED>(p, n, y[0], y[S - 1]));
    }
}

// Many rows of x: a workgroup of WN x WM wavefronts has 32 HN WN rows of weights (two halves: of gate and of up, where gated) and 16 MT WM rows
// of x.  EVEN: all rows of a half have one block's scale.  A block of the width is 128 bytes of each row, copied to LDS STAGES - 1 blocks ahead; piece p of row r lies at place
// p ^ (r & 7), so that eight lanes reading one piece of eight rows touch all banks.
// 256 x 256 results take 2048 cycles a block of the matrix units, as many of the copies (a CU gets 32 bytes a cycle from L2), and 2300 of
// a SIMD's issue slots (a product takes 16 of its 32 cycles', the 160 other vector instructions 4 each); together about 2750, at 1.8 GHz: the clock
// falls with the matrix units' load.  4096 x 12288 x 4096 161 us (2.56 PFLOP/s; 170 on one machine), gated 4096 x 4096 x 2 x 12288 336 us (2.45; 363), 4096 x 4096 x 4096
// 56.7 us; nine vector instructions fewer with moving descriptors instead, 166 us for 162.
template <int DT, int HN, int MT, int WN, int WM, int STAGES, bool EVEN, bool GATED>
__global__ void __launch_bounds__(64 * WN * WM) product_many_kernel(const ProductParams p) {
    constexpr int kWaves = WN * WM, kHalf = 16 * HN * WN, kX = 16 * MT * WM;
    constexpr int kScales = (2 * kHalf + kX) * 128, kStage = kScales + 4 * kX + 256;      // codes, scales of x, of each unit of weights
    constexpr int kScaleCopies = (kX / 64 + kWaves) / kWaves;
    constexpr int kHalfCopies = kHalf / 8 / kWaves, kXCopies = kX / 8 / kWaves;          // of 8 rows, a wavefront
    static_assert(128 % kHalf == 0 && kHalf % (8 * kWaves) == 0 && kX % (8 * kWaves) == 0 && kX % 64 == 0 && 2 * kHalf <= 16 * 64, "whole copies");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * kStage];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r = lane & 15u, g = lane >> 4;
    // Workgroups go to the eight XCDs in turn: each takes a run of neighbouring tiles, six rows of tiles wide, which is nearly
    // square for the 32 it has at once, and its L2 holds their rows.
    constexpr uint32_t kN = GATED ? kHalf : 2 * kHalf;     // results a workgroup
    const uint32_t tiles_n = (p.cols + kN - 1u) / kN, tiles_m = (p.rows + kX - 1u) / kX;
    const uint32_t at = (blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (at >= tiles_n * tiles_m) return;
    const uint32_t band = at / (6u * tiles_n), in_band = at - band * 6u * tiles_n, deep = min(6u, tiles_m - 6u * band);
    const uint32_t tile_n = __builtin_amdgcn_readfirstlane(in_band / deep), tile_m = __builtin_amdgcn_readfirstlane(6u * band + (in_band - tile_n * deep));
    const uint32_t n0 = tile_n * kN, m0 = tile_m * kX;
    const uint32_t w_rows = (GATED ? 2u : 1u) * p.cols;
    const uint32_t first[2] = {n0, n0 + (GATED ? p.cols : (uint32_t)kHalf)};
    u32x4_t wr[2];
    wr[0] = tile_words(p.w, p.w_row, first[0], p.cols, kHalf, p.width);
    wr[1] = tile_words(p.w, p.w_row, first[1], w_rows, kHalf, p.width);
    const u32x4_t xr = tile_words(p.x, p.x_row, m0, p.rows, kX, p.width);
    const uint32_t wn = wave % WN, wm = wave / WN;
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(lds);
    const uint32_t piece = 16u * ((lane & 7u) ^ (lane >> 3));
    const uint32_t w_off = (wave * kHalfCopies * 8u + (lane >> 3)) * (uint32_t)p.w_row + piece, x_off = (wave * kXCopies * 8u + (lane >> 3)) * (uint32_t)p.x_row + piece;
    constexpr int kUnits = 2 * HN;
    // Scales: 64 rows of x a copy, then one of the weights', a number for each 16 rows.  A wavefront has one copy or more of either kind (a copy
    // too many repeats the weights'): no branch in the loop, past which the compiler would move the sums.
    uint32_t scale_off[kScaleCopies];
    uint64_t scale_base[kScaleCopies], scale_step[kScaleCopies];
#pragma unroll
    for (int c = 0; c < kScaleCopies; c++) {
        const uint32_t t = wave + (uint32_t)(c * kWaves), u = min(lane, 2u * kHalf / 16u - 1u), h = u / (kHalf / 16u);
        scale_off[c] = t < kX / 64u ? 4u * (min(m0 + 64u * t + lane, p.rows - 1u) - m0) * (uint32_t)p.xs_row
                                    : 4u * (min((h ? first[1] : first[0]) + 16u * (u - h * (kHalf / 16u)), w_rows - 1u) / 128u) * (uint32_t)p.ws_row;
        scale_base[c] = t < kX / 64u ? reinterpret_cast<uintptr_t>(p.x_scale + (int64_t)m0 * p.xs_row) : reinterpret_cast<uintptr_t>(p.w_scale);
        scale_step[c] = 4u * (uint64_t)(t < kX / 64u ? p.xs_col : p.ws_col);
        asm("" : "+s"(scale_base[c]), "+s"(scale_step[c]));              // (in registers: not to be chosen again each time)
    }
    const uint32_t last = p.blocks - 1u;
    // Copy q of a wavefront's kCopies of block b (behind the last block: zeroes, from no memory).
    constexpr int kCopies = kScaleCopies + 2 * kHalfCopies + kXCopies;
    // With two stages, the copies of x and the scales start as soon as all wavefronts have theirs in registers, behind a barrier of their own in
    // the first units, and those of the weights behind the last unit: something is always on its way.
    constexpr bool kEarly = STAGES == 2;
    constexpr int kWCopies = 2 * kHalfCopies, kEarlyCopies = kCopies - kWCopies;
    static_assert(kEarly ? kWCopies <= MT && kEarlyCopies <= MT * (kUnits - 2) : kCopies >= MT && kCopies <= MT * kUnits, "a place for each copy");
    static_assert((STAGES - 2) * kCopies < 64 && kEarlyCopies < 64, "a count of six bits");
    auto copy_part = [&](uint32_t b, uint32_t stage, int q) {
        const uint32_t k = 128u * b, base = lds0 + stage * kStage;
        const bool inside = k + piece < p.width;           // (a multiple of 16)
        if (q < kScaleCopies) {
            const uint32_t t = wave + (uint32_t)(q * kWaves);
            const uint64_t a = scale_base[q] + min(b, last) * scale_step[q];
            copy_word((u32x4_t){(uint32_t)a, (uint32_t)(a >> 32) & 0xFFFFu, 0x7FFFFFFFu, 0x00020000u}, base + kScales + (t < kX / 64u ? 256u * t : 4u * kX), scale_off[q]);
        } else if (q < kScaleCopies + 2 * kHalfCopies) {
            const int h = (q - kScaleCopies) / kHalfCopies, t = (q - kScaleCopies) % kHalfCopies;
            copy_piece(wr[h], base + (h * kHalf + (wave * kHalfCopies + t) * 8) * 128, inside ? w_off + 8u * t * (uint32_t)p.w_row + k : kNowhere);
        } else {
            const int t = q - kScaleCopies - 2 * kHalfCopies;
            copy_piece(xr, base + (2 * kHalf + (wave * kXCopies + t) * 8) * 128, inside ? x_off + 8u * t * (uint32_t)p.x_row + k : kNowhere);
        }
    };
    auto copy_early = [&](uint32_t b, uint32_t stage, int i) { copy_part(b, stage, i < kScaleCopies ? i : i + kWCopies); };
    f32x4 acc[2][HN][MT];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < HN; i++)
#pragma unroll
            for (int j = 0; j < MT; j++) acc[h][i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const uint32_t read0 = r * 128u + 16u * (g ^ (r & 7u));
    auto read_rows = [&](uint32_t stage, uint32_t row) -> i32x8 {
        const uint8_t *q = lds + stage * kStage + row * 128u;
        const u32x4_t lo = *reinterpret_cast<const u32x4_t *>(q + read0), hi = *reinterpret_cast<const u32x4_t *>(q + (read0 ^ 64u));
        return (i32x8){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
    // Unit u is 16 rows of weights with all of the wavefront's x.  Its products start while the sums of the unit before are scaled and added
    // and the codes of the next are on their way from LDS: a product of 32 cycles, then the five instructions for an earlier one.  The next
    // block is waited for in front of the last unit, whose codes are in registers by then, and read beneath its products.
    i32x8 xv[MT], wq[2];
    f32x4 d[MT];
    constexpr int kW = EVEN ? 2 : kUnits, kPerW = kUnits / kW;
    float xn[MT], wv[kW], late[MT];                        // scales of this block, of the last unit's sums
    auto read_unit = [&](uint32_t stage, int u) { wq[u & 1] = read_rows(stage, (u / HN) * kHalf + 16u * (wn * HN + u % HN)); };
    auto add = [&](int u, int j, f32x4 v, float f) {
#pragma unroll
        for (int e = 0; e < 4; e++) acc[u / HN][u % HN][j][e] = fmaf(v[e], f, acc[u / HN][u % HN][j][e]);
    };
    auto read_scales = [&](uint32_t stage) {
        const float *q = reinterpret_cast<const float *>(lds + stage * kStage + kScales);
#pragma unroll
        for (int j = 0; j < MT; j++) xn[j] = q[16u * (wm * MT + j) + r];
#pragma unroll
        for (int u = 0; u < kUnits; u += kPerW) wv[u / kPerW] = q[kX + (u / HN) * (kHalf / 16) + wn * HN + u % HN];
    };
#pragma unroll
    for (int b = 0; b + (kEarly ? 0 : 1) < STAGES; b++)
#pragma unroll
        for (int q = 0; q < kCopies; q++) copy_part(b, b, q);
    copies_but<(kEarly ? 1 : STAGES - 2) * kCopies>();
    if (!kEarly) {
#pragma unroll
        for (int q = 0; q < MT; q++) copy_part(STAGES - 1, STAGES - 1, q);
    }
    read_scales(0);
    read_unit(0, 0);
#pragma unroll
    for (int j = 0; j < MT; j++) {
        xv[j] = read_rows(0, 2u * kHalf + 16u * (wm * MT + j));
        d[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        late[j] = 0.f;
    }
    uint32_t stage = 0, before = STAGES - 1;               // of this block, of the one in front of it (where the block STAGES - 1 behind it goes)
    for (uint32_t b = 0; b < p.blocks; b++) {
        const uint32_t next = stage + 1 == STAGES ? 0u : stage + 1u;
#pragma unroll
        for (int u = 0; u < kUnits - 1; u++) {
            read_unit(stage, u + 1);
            __builtin_amdgcn_sched_barrier(0);             // (left to itself the compiler puts each sum right behind its product, and waits)
#pragma unroll
            for (int j = 0; j < MT; j++) {
                const f32x4 v = d[j];
                d[j] = block_product(wq[u & 1], xv[j]);
                if (u) add(u - 1, j, v, xn[j] * wv[(u - 1) / kPerW]);
                else add(kUnits - 1, j, v, late[j]);
                if (kEarly ? u >= 1 && MT * (u - 1) + j < kEarlyCopies : MT * (u + 1) + j < kCopies) {
                    if (kEarly) copy_early(b + STAGES, stage, MT * (u - 1) + j);
                    else copy_part(b + (STAGES - 1), before, MT * (u + 1) + j);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (kEarly && u == 0) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        float f[MT];
#pragma unroll
        for (int j = 0; j < MT; j++) {
            f[j] = xn[j] * wv[(kUnits - 2) / kPerW];
            late[j] = xn[j] * wv[kW - 1];
        }
        copies_but<kEarly ? kEarlyCopies : (STAGES - 2) * kCopies>();              // the next block is there (behind the last one, what is read below is not used)
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const f32x4 v = d[j];
            d[j] = block_product(wq[1], xv[j]);
            if (kEarly ? j < kWCopies : true) copy_part(b + STAGES, stage, kEarly ? kScaleCopies + j : j);          // (one at a time, as it is sent)
            if (j == 0) read_unit(next, 0);
            xv[j] = read_rows(next, 2u * kHalf + 16u * (wm * MT + j));
            add(kUnits - 2, j, v, f[j]);
            if (j + 1 == MT) read_scales(next);
            __builtin_amdgcn_sched_barrier(0);
        }
        before = stage;
        stage = next;
    }
    copies_done();                                         // (nothing may arrive in LDS that another workgroup has by then)
#pragma unroll
    for (int j = 0; j < MT; j++) add(kUnits - 1, j, d[j], late[j]);
    // A lane has four neighbouring results of a row.  Through LDS, each wavefront in a part of its own, the rows' pieces are put together to whole
    // lines: stored as they are, 4096 x 4096 results take 14 us, so 5.  Pieces that are not there go nowhere, without a branch (with one a store,
    // 4096 x 4096 x 12288 178 us, so 167.6); a row of tiles at once where it fills lines, or all of the wavefront's (4096 x 4096 x 4096 56.7 us and 57.4;
    // 512 x 4096 x 6144, half lines, 19.2 and 18.9).
    constexpr int kRow = 32 * HN, kPitch = kRow + 16, kLanes = kRow / 16, kRows = 64 / kLanes;       // bytes, lanes of a row, rows of a store
    constexpr int kSlice = HN == 4 ? 1 : MT;               // of 16 rows
    static_assert(kWaves * 16 * kSlice * kPitch <= STAGES * kStage, "room for the results");
    uint8_t *own = lds + wave * (16 * kSlice * kPitch);
    const uint32_t m_w = m0 + 16u * MT * wm, pitch = 2u * (uint32_t)p.out_row;
    const auto out = __builtin_amdgcn_make_buffer_rsrc(p.out + (int64_t)m_w * p.out_row, 0, (int)(m_w < p.rows ? min(p.rows - m_w, 16u * MT) * pitch : 0u), 0x00020000);
#pragma unroll
    for (int h = 0; h < (GATED ? 1 : 2); h++) {
        const uint32_t n_h = first[h] + 16u * (wn * HN), n_l = n_h + 8u * (lane % kLanes), off = n_l < p.cols ? lane / kLanes * pitch + 2u * n_l : kNowhere;
#pragma unroll
        for (int j0 = 0; j0 < MT; j0 += kSlice) {
#pragma unroll
            for (int i = 0; i < HN; i++)
#pragma unroll
                for (int j = j0; j < j0 + kSlice; j++) {
                    const uint32_t m = m0 + 16u * (wm * MT + j) + r, n = n_h + 16u * i + 4u * g;
                    const u32x2 v = four_results<DT, GATED>(p, n, acc[h][i][j], acc[1][i][j]);
                    if (p.whole8) *reinterpret_cast<u32x2 *>(own + (16 * (j - j0) + r) * kPitch + 32 * i + 8 * g) = v;
                    else if (m < p.rows && n < p.cols) store_four(p, m, n, v);
                }
            if (!p.whole8) continue;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // (the wavefront's own: no barrier)
#pragma unroll
            for (int t = 0; t < 16 * kSlice / kRows; t++) {
                const u32x4_t v = *reinterpret_cast<const u32x4_t *>(own + ((uint32_t)(t * kRows) + lane / kLanes) * kPitch + 16u * (lane % kLanes));
                const uint32_t to = off + (16u * j0 + (uint32_t)(t * kRows)) * pitch;
                if (p.past) __builtin_amdgcn_raw_buffer_store_b128(v, out, to, 0, 2);
                else __builtin_amdgcn_raw_buffer_store_b128(v, out, to, 0, 0);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
}

static int check_launch(const ProductParams &p, uint64_t threads) {
    PKV_REQUIRE(threads < (1ull << 32), PKV_ERR_UNSUPPORTED, "rows x results too large");
    PKV_REQUIRE(apart(p.rows, p.out_row, p.cols, 1), PKV_ERR_INVALID, "results must not overlap");
    return PKV_OK;
}
template <int DT, bool GATED, int RT, int MT> int launch_few(const ProductParams &p, hipStream_t s) {
    const uint64_t tiles = (uint64_t)((p.cols + 16 * RT - 1) / (16 * RT)) * ((p.rows + 16 * MT - 1) / (16 * MT)), wgs = (tiles + 7) / 8 * 8;
    if (const int rc = check_launch(p, wgs * 512)) return rc;
    product_few_kernel<DT, RT, MT, GATED><<<dim3((unsigned)wgs), 512, 0, s>>>(p);
    PKV_HIP_CHECK(hipGetLastError());
    return PKV_OK;
}
template <int DT, bool GATED, int HN, int MT, int WN, int WM, int STAGES> int launch_many(const ProductParams &p, hipStream_t s) {
    constexpr uint64_t n = (GATED ? 16 : 32) * HN * WN, m = 16 * MT * WM;
    const uint64_t tiles = (p.cols + n - 1) / n * ((p.rows + m - 1) / m), wgs = (tiles + 7) / 8 * 8;
    if (const int rc = check_launch(p, wgs * (64 * WN * WM))) return rc;
    // (a half of a tile's rows of weights may have two blocks of 128, and two scales, only where up's rows start within one)
    if (!GATED || p.cols % (16 * HN * WN) == 0) product_many_kernel<DT, HN, MT, WN, WM, STAGES, true, GATED><<<dim3((unsigned)wgs), 64 * WN * WM, 0, s>>>(p);
    else if constexpr (GATED) product_many_kernel<DT, HN, MT, WN, WM, STAGES, false, GATED><<<dim3((unsigned)wgs), 64 * WN * WM, 0, s>>>(p);
    PKV_HIP_CHECK(hipGetLastError());
    return PKV_OK;
}
// Which workgroup a product gets: the one with the shortest estimate
//     max(bytes of w / 6.4 TB/s, rounds of 256 workgroups * (blocks of the width * us a block + us a round)),
// both times a shape's own, fitted to 125 products of 1 to 4096 rows, 896 to 12288 wide, 1024 to 24576 rows of w (0.2 % slower in the mean than the
// best shape of each, 6 % at most).  What that is about, us: 48 x 4096 x 6144, 32 x 48 results a workgroup 7.9, 64 x 64 10.7, 128 x 64 13; 512 x 4096 x 6144,
// 64 x 64 27.4, 128 x 128 20.5; 1024 x 4096 x 6144, 128 x 128 33.8, 128 x 256 30.8; 2048 x 4096 x 6144, 128 x 128 60, 256 x 256 49; one row of 4096 x 1024,
// 16 x 16 3.6, 32 x 32 5.1.
struct Shape {
    int rt, mt;                          // tiles of 16 results: of w (of gate and up each half as many, from 128 results on), of x
    float block_us, round_us;
};
constexpr Shape kShapes[] = {{1, 1, .048f, .3f},  {1, 2, .068f, .5f},  {2, 2, .098f, .7f},  {2, 3, .133f, 1.1f},  {4, 2, .133f, 1.5f}, {4, 3, .155f, 2.f},
                             {4, 4, .184f, 2.5f}, {8, 4, .377f, 1.1f}, {8, 8, .521f, 1.3f}, {8, 16, .855f, 3.f}, {16, 16, 1.46f, 4.3f}};
template <int DT, bool GATED> int launch_product(const ProductParams &p, hipStream_t s) {
    const double stream_us = (double)p.width * p.cols * (GATED ? 2 : 1) / 6.4e6;
    double least = 0.;
    uint64_t rounds_of = 0;
    int best = -1;
    for (int i = 0; i < (int)(sizeof kShapes / sizeof kShapes[0]); i++) {
        const Shape &h = kShapes[i];
        const bool many = h.rt >= 8;
        if (GATED && h.rt == 4) continue;                  // (32 tiles of sums and their codes: not in registers and LDS together)
        const uint64_t n = 16u * h.rt / (GATED && many ? 2 : 1), m = 16u * h.mt;
        const uint64_t rounds = ((p.cols + n - 1) / n * ((p.rows + m - 1) / m) + 255) / 256;
        double block = h.block_us, round = h.round_us;
        if (GATED && !many) block *= 1.3 * (2 * h.rt + h.mt) / (h.rt + h.mt);
        if (h.rt == 8 && h.mt == 8 && rounds == 1) { block = .54; round = 1.8; }         // (four stages, one workgroup a CU: below)
        const double us = (double)rounds * (p.blocks * block + round), t = us > stream_us ? us : stream_us;
        if (best < 0 || t < least) { least = t; best = i; rounds_of = rounds; }
    }
    switch (best) {
    case 0: return launch_few<DT, GATED, 1, 1>(p, s);
    case 1: return launch_few<DT, GATED, 1, 2>(p, s);
    case 2: return launch_few<DT, GATED, 2, 2>(p, s);
    case 3: return launch_few<DT, GATED, 2, 3>(p, s);
    case 4: if constexpr (!GATED) return launch_few<DT, GATED, 4, 2>(p, s);
    case 5: if constexpr (!GATED) return launch_few<DT, GATED, 4, 3>(p, s);
    case 6: if constexpr (!GATED) return launch_few<DT, GATED, 4, 4>(p, s);
    // Stages: as many as leave two workgroups a CU where there are that many (64 rows, three of 25 KB: 256 x 2048 x 8192 10.2 us, with six 11.2), as LDS
    // holds where there is one (128 x 128: 512 x 2048 x 8192 with two 17.7 us, with four 14.8; 2048 x 4096 x 6144, twice as many: 67, 70).
    case 7: return launch_many<DT, GATED, 2, 1, 2, 4, 3>(p, s);
    case 8: return rounds_of > 1 ? launch_many<DT, GATED, 2, 2, 2, 4, 2>(p, s) : launch_many<DT, GATED, 2, 2, 2, 4, 4>(p, s);
    case 9: return launch_many<DT, GATED, 2, 4, 2, 4, 3>(p, s);
    default: return launch_many<DT, GATED, 4, 4, 2, 4, 2>(p, s);
    }
}

}  // namespace pkv

extern "C" int pkv_fp8_product(const pkv_fp8_product_args *a, pkv_stream_t s_) {
    using namespace pkv;
    hipStream_t s = (hipStream_t)s_;
    PKV_REQUIRE(a && a->x && a->w && a->x_scale && a->w_scale && a->out, PKV_ERR_INVALID, "null pointer argument");
    PKV_REQUIRE(a->dtype == PKV_F16 || a->dtype == PKV_BF16, PKV_ERR_UNSUPPORTED, "Unsupported data type");
    PKV_REQUIRE(a->rows > 0 && a->width > 0 && a->cols > 0, PKV_ERR_INVALID, "sizes must be positive");
    PKV_REQUIRE(a->width % 16 == 0 && a->width <= (1 << 20), PKV_ERR_UNSUPPORTED, "not supported: width %d (multiples of 16 up to 2^20)", a->width);
    PKV_REQUIRE(a->rows <= (1 << 24) && a->cols <= (1 << 24), PKV_ERR_UNSUPPORTED, "not supported: more than 2^24 rows or results");
    PKV_REQUIRE(!a->gated || (a->cols % 16 == 0 && !a->bias), PKV_ERR_UNSUPPORTED, "not supported: a gated product of %d results (multiples of 16, no bias)", a->cols);
    PKV_REQUIRE((((uintptr_t)a->x | (uintptr_t)a->w | (uintptr_t)a->x_stride | (uintptr_t)a->w_stride) % 16) == 0, PKV_ERR_INVALID,
                "rows must start on 16-byte boundaries");
    PKV_REQUIRE(((uintptr_t)a->x_scale | (uintptr_t)a->w_scale) % 4 == 0 && ((uintptr_t)a->bias | (uintptr_t)a->out) % 2 == 0, PKV_ERR_INVALID,
                "scales, bias and results must lie at multiples of their size");
    PKV_REQUIRE(a->x_scale_stride[0] >= 0 && a->x_scale_stride[0] <= (1 << 20) && a->w_scale_stride[0] >= 0 && a->w_scale_stride[0] <= (1 << 20) &&
                (uint64_t)a->w_scale_stride[0] * (uint64_t)((a->gated ? 2 : 1) * (int64_t)a->cols / kBlock8 + 1) < (1u << 29), PKV_ERR_UNSUPPORTED,
                "not supported: scales of neighbouring rows more than 2^20 apart, or of w over 2 GiB");
    // (a row that overlaps the next is one that the caller repeats: stride 0)
    PKV_REQUIRE((a->x_stride == 0 || a->x_stride >= a->width) && a->x_stride <= (1 << 20) && a->w_stride >= 0 && a->w_stride <= (1 << 20) &&
                (a->w_stride == 0 || a->w_stride >= a->width), PKV_ERR_UNSUPPORTED, "not supported: rows of x or w more than 2^20 bytes apart, or that overlap");
    ProductParams p;
    p.x = a->x; p.w = a->w; p.x_scale = a->x_scale; p.w_scale = a->w_scale; p.bias = (const uint16_t *)a->bias; p.out = (uint16_t *)a->out;
    p.x_row = a->x_stride; p.w_row = a->w_stride; p.out_row = a->rows > 1 ? a->out_stride : a->cols;            // (one row's stride means nothing)
    p.xs_row = a->x_scale_stride[0]; p.xs_col = a->x_scale_stride[1]; p.ws_row = a->w_scale_stride[0]; p.ws_col = a->w_scale_stride[1];
    p.rows = (uint32_t)a->rows; p.width = (uint32_t)a->width; p.cols = (uint32_t)a->cols;
    p.blocks = (p.width + kBlock8 - 1) / kBlock8;
    p.whole4 = (p.cols | (uint64_t)p.out_row) % 4 == 0 && (uintptr_t)a->out % 8 == 0;
    // Results that no L2 would hold until they are read: 1024 x 128 x 6144 (12.6 MB) 7.5 -> 6.7 us, 4096 x 4096 x 4096 (33.5 MB) 59.5 -> 58.2.
    p.past = (uint64_t)p.rows * p.cols * 2u > (4u << 20);
    p.whole8 = (p.cols | (uint64_t)p.out_row) % 8 == 0 && (uintptr_t)a->out % 16 == 0 && p.out_row >= 0 && p.out_row <= (1 << 23);       // (64 rows within 2^30 bytes)
    if (a->gated) return a->dtype == PKV_F16 ? launch_product<PKV_F16, true>(p, s) : launch_product<PKV_BF16, true>(p, s);
    return a->dtype == PKV_F16 ? launch_product<PKV_F16, false>(p, s) : launch_product<PKV_BF16, false>(p, s);
}
