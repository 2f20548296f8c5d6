// Attention of several new tokens over a compressed cache: query i of n sits at position T - n + i of the T tokens (streams, then
// the 16-bit window) and attends to those from the sequence's first token up to itself.
//
// Rows are the (token, query head) pairs of one KV head, row = token * G + head of the group: a workgroup takes RG groups of 32 NB of
// them and a run of 128-token tiles; each of a group's four wavefronts takes 32 tokens of every tile for ALL of the group's rows and
// keeps a softmax state and an accumulator of its own, so nothing of the softmax crosses wavefronts until the run ends.
//
// Both products are formed transposed, on 32x32x16 fp16 matrix instructions (a product's columns are the lanes, here the rows):
//   S^T [token x row]   = K codes x q      a lane holds 16 tokens' scores of one row: maxima and sums are the lane's own but for
//                                          one exchange with lane ^ 32, and exp2's results are the next product's operand as they lie
//   O^T [channel x row] = V codes x p      the factor of a new maximum is a number of the lane
// Codes enter as whole numbers in fp16: 0x6400 | code is 1024 + code, and one packed subtraction takes the 1024 away.  (The integer
// itself, read as a half, is the code times 2^-24 and needs no subtraction, but the matrix cores add up products of subnormals
// without normalising them, to about 18 bits.)  Scale and zero of a token are applied to what the products need of them, in fp32:  score = scale (q . code + zero sum(q)),
// out = sum p scale code + sum p scale zero.  The weight p * scale is rounded to fp16, scaled by a power of two that follows
// the largest scale met: by 2^-11 of it, or 2^-31 of the largest scale that the row sees where that is more; the zero's sum takes the
// rounded weight, so that the error is 2^-11 of p |v|, not of p * scale * code.  Where a row does not see all that was met, its weights
// follow what it sees (unseen_shift; 1 to 2 % of a prompt's time, 116 us to 118 for 2048 queries on 2048 tokens).
// p is taken against a maximum that is raised only once a score exceeds it by 2^8 (weights stay below 2^15): the factor on the
// accumulators, and the exchange of maxima between lanes, are rare, and the reference goes into the scores' own multiply-add.
// q in bf16 becomes fp16 times one power of two for the workgroup's rows, or one of each row's own where they lie 2^8 apart or more, which
// loses bits only of values 2^-20 below their row's largest (where fp16 has no normal numbers left; rows up to 2^100 apart).  The branch
// for such rows costs the others up to 3 % (1024 queries over 16384 tokens 522 -> 539 us, 8 x 8 over 16384 none).
//
// K turns through LDS (a pack holds 16 tokens of one channel, the product wants channels of one token): codes as bytes in rows of
// 136 bytes, private to the wavefront.  V needs no turn: lane = channel, and the order of the tokens in the contraction is free as
// long as both operands agree, so a lane unpacks ONE pack per 32 channels straight into its operand -- tokens (k, k + 8) side by
// side, since both halves of a pack's word take the same shifts.  Which pack is where comes from a table that the half-wavefronts
// fill, one unit each (offset, width, minimum of its 128 packs).
//
// Bound by the vector instructions around the products: 32 tokens take a wavefront some 770 of them with 32 rows (of a tile: K's codes
// to bytes 210, bytes to operands 65, V's table 80 and packs 180, scores to weights 150), 70 less with 16, 730 with 64.  Hence as few
// wavefronts as possible unpack the same block, up to 128 rows a workgroup, two groups of them sharing K's bytes and V's table; and
// three workgroups a CU where rows are few (vector units busy 79 % of the cycles, 67 % with two).  8 KV heads, 4-bit codes: 8 sequences
// x 4 queries of 32 heads over 16384 tokens 69 us (79 with two workgroups a CU, 74 with products of 32 rows; a copy of the bytes: 22),
// 1024 queries over 32768 1015 us, 540 TFLOP/s (a large product reaches 1160), where 64 rows a workgroup without sharing took 1430;
// 40 heads x 333 queries of two sequences over 4096 tokens in 5-bit codes 138 to 171 us, by their padding; 3 queries over 1100 tokens 13 us, 4 of them the
// merge.
#include "pkv_block.hpp"
#include "pkv_runtime.hpp"

namespace pkv {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kChunkTile = 128;
constexpr int kKRow = 136;                     // bytes of a token's K codes in LDS: 34 dwords, 32 rows start at 32 different banks
constexpr int kQRow = 272;                     // bytes of a row of q: 68 dwords
constexpr int kVRow = 264;                     // bytes of a window token's V
constexpr int kPart = 132;                     // floats of a partial: maximum, sum, 2 unused, 128 channels
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.0e38f;            // a maximum before any score; a masked score is -inf, so its weight is 0 against it

struct ChunkParams {
    const uint8_t *k_stream, *v_stream;
    const uint32_t *k_info, *v_info;
    const uint16_t *k_scale, *k_zero, *v_scale, *v_zero, *k_win, *v_win, *q;
    uint16_t *out;
    float *part;                               // NULL: one run, the result is written
    const int32_t *starts;
    int64_t q_b, q_h, q_t, o_b, o_h, o_t;
    uint64_t k_bytes, v_bytes;
    int Hq, Hkv, BH, G, n, rows, T_c, T_w, par_stride, win_stride, k_bits, v_bits, causal;
    int tiles_c, tiles, run, nsplit, row_tiles;
    uint32_t slot_k, slot_v, ring;             // LDS bytes of a staged block of either side and of everything staged
    float sm_log2;
};

__device__ __forceinline__ float chunk_f32(uint32_t bits16, bool bf) {
    return bf ? __uint_as_float(bits16 << 16) : __half2float(__ushort_as_half((unsigned short)bits16));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, (h2v){(_Float16)a, (_Float16)b});
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, b2));
}
template <bool BF> __device__ __forceinline__ f16v product(u4 a, u4 b, f16v c) {
    if (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

template <bool BF> __device__ __forceinline__ f4v product16(u4 a, u4 b, f4v c) {
    if (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Two of four codes (one a byte) as halves.
__device__ __forceinline__ uint32_t codes_f16(uint32_t c4, uint32_t which) {
    return __builtin_bit_cast(uint32_t, (h2v)(__builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, c4, which)) - (h2v){(_Float16)1024.f, (_Float16)1024.f}));
}

// The eight operand registers of one V pack (table entry e: LDS address | width << 17 | minimum << 21): tokens (j, j + 8) side by
// side, j = 0..7.  The field, 1024 + (code - minimum), and minimum - 1024 add up exactly.
__device__ __forceinline__ uint32_t field_code(uint32_t shifted, uint32_t mask, h2v low) {
    return __builtin_bit_cast(uint32_t, (h2v)(__builtin_bit_cast(h2v, (shifted & mask) | 0x64006400u) + low));
}
template <bool WIDE> __device__ __forceinline__ void pack_operand(const uint8_t *ring, uint32_t e, uint32_t out[8]) {
    typedef unsigned short u16pair __attribute__((ext_vector_type(2)));
    const uint32_t at = e & 0x1FFFFu, len = (e >> 17) & 15u;
    const uint32_t mask = ((1u << len) - 1u) * 0x00010001u;
    const h2v low = __builtin_bit_cast(h2v, 0x64006400u | ((e >> 21) * 0x00010001u)) - (h2v){(_Float16)2048.f, (_Float16)2048.f};
    if (WIDE) {                                // words of up to 128 bits: two tokens at a time, bits (14 - j) * len of the word on
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            uint32_t win[2];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t bit = (uint32_t)(14 - 8 * half - j) * len, byte = at + (bit >> 3);
                const uint32_t *d = reinterpret_cast<const uint32_t *>(ring + (byte & ~3u));
                win[half] = __builtin_amdgcn_alignbyte(d[1], d[0], byte & 3u) >> (bit & 7u);
            }
            const u16pair w = __builtin_bit_cast(u16pair, __builtin_amdgcn_perm(win[1], win[0], 0x05040100u));
            out[j] = field_code(__builtin_bit_cast(uint32_t, (u16pair)(w >> __builtin_bit_cast(u16pair, len * 0x00010001u))), mask, low);
            out[j + 1] = field_code(__builtin_bit_cast(uint32_t, w), mask, low);
        }
        return;
    }
    const uint64_t word = lds_load64(ring, at);
    const uint32_t hi = (uint32_t)(word >> (8u * len)), lo = (uint32_t)word;       // tokens 0..7 | 8..15
    const u16pair w[2] = {__builtin_bit_cast(u16pair, __builtin_amdgcn_perm(lo >> (4u * len), hi >> (4u * len), 0x05040100u)),
                          __builtin_bit_cast(u16pair, __builtin_amdgcn_perm(lo, hi, 0x05040100u))};
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const u16pair sh = __builtin_bit_cast(u16pair, len * (uint32_t)(3 - (j & 3)) * 0x00010001u);
        out[j] = field_code(__builtin_bit_cast(uint32_t, (u16pair)(w[j >> 2] >> sh)), mask, low);
    }
}

// Widths, minima and places (bytes from the unit's start) of the lane's four packs, for codes of up to 4 bits.
__device__ __forceinline__ void narrow_packs(const uint8_t *unit, int t, const UnitGeom g, uint32_t len[4], uint32_t mn[4], uint32_t at[4]) {
    const uint32_t minsw = lds_meta_word(unit, t, g.W), lensw = lds_meta_word(unit + g.mins_bytes, t, g.LB);
    uint32_t off2[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        len[i] = (lensw >> (i * g.LB)) & ((1u << g.LB) - 1u);
        mn[i] = (minsw >> (i * g.W)) & ((1u << g.W) - 1u);
    }
    pack_offsets8(len[0] | (len[1] << 8) | (len[2] << 16) | (len[3] << 24), off2);        // (widths of 7, damaged, do not carry either)
#pragma unroll
    for (int i = 0; i < 4; i++) at[i] = (uint32_t)(g.mins_bytes + g.lens_bytes) + 2u * off2[i];
}

// Blocks travel from memory to LDS without registers (but for wide codes where rows are few), 16 bytes a lane: lane l's land at lds_addr + 16 l, lanes behind
// the buffer's end get zeroes, lanes that are off write nothing.  lds_addr and rsrc are wave-uniform.  The compiler does not see the
// copies: s_waitcnt vmcnt(0) stands in front of the barrier that hands them on, and the barrier between waits for LDS only.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy_to_lds(u4 rsrc, uint32_t lds_addr, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(lds_addr), "v"(voff), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop

// The largest of the wavefront's values, in every lane (the upper half of the lanes repeats the lower).
__device__ __forceinline__ uint32_t half_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, true));
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 31);
}

// One 32-row block's softmax step for 16 scores of the lane's row: the new maximum, the factor for what was summed before, and the
// weights in place of the scores.
__device__ __forceinline__ float softmax_step(f16v &y, float &m) {
    float top = y[0];
#pragma unroll
    for (int r = 1; r < 16; r++) top = fmaxf(top, y[r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float was = m;
    m = fmaxf(m, top);
#pragma unroll
    for (int r = 0; r < 16; r++) y[r] = __builtin_amdgcn_exp2f(y[r] - m);
    return __builtin_amdgcn_exp2f(was - m);
}

// A row that sees only some of a wavefront's 32 tokens: the power of two (at most 2^80) by which its reference goes down, so that its
// weights follow the largest V scale of what it sees and not of the tokens behind.  most: that of the 32 as written (2^6 .. 2^7 for the
// largest of all tokens met); past: that of the tokens before, 0 if there are none; sum: its sum of weights, which stays below 2^101.
__device__ __forceinline__ float unseen_shift(float most, float past, float sum) {
    const int e = (int)(__float_as_uint(fmaxf(most, past)) >> 23), room = 227 - (int)(__float_as_uint(sum) >> 23);
    return e ? (float)max(min(min(133 - e, 80), room), 0) : 0.f;
}

template <bool BF, int NB, int RG, bool WIDE, bool R16 = false>
__global__ void __launch_bounds__(256 * RG, RG == 2 ? 1 : WIDE ? 2 : 3) attn_chunk_kernel(const ChunkParams p) {
    constexpr int NQ = WIDE ? 9 : 5;                       // 1 KiB steps that hold a staged block
    constexpr bool ONCE = RG == 1 && !WIDE;                // a tile's blocks are staged one at a time
    static_assert(!R16 || (ONCE && NB == 1), "sixteen rows: one workgroup's, narrow codes");
    constexpr int M = R16 ? 16 : 32 * NB * RG, kKBufs = ONCE ? 1 : 2, kBufs = ONCE ? 1 : RG + 1, kSets = RG;
    constexpr bool COPY = !WIDE || RG == 2;                // blocks go to LDS without registers (what is staged lies below 64 KiB)
    extern __shared__ __align__(16) uint8_t lds[];
    uint8_t *ring = lds;                                   // staged: kKBufs tiles' K blocks, kBufs tiles' V blocks; window and end: V rows, sums (kt as well)
    uint8_t *kt_all = lds + p.ring;                        // [kSets][4 quarters][32 tokens][kKRow]
    uint32_t *tab_all = reinterpret_cast<uint32_t *>(kt_all + kSets * 4 * 32 * kKRow);        // [kSets][8 units][4 slots][32 lanes]
    float2 *par_all = reinterpret_cast<float2 *>(tab_all + kSets * 1024);          // [kSets][2][4][32]: (scale, zero * scale), (V scale, V zero)
    float *st = reinterpret_cast<float *>(par_all + kSets * 256);                  // [2][4][M] maxima, sums at the end
    uint8_t *qt = reinterpret_cast<uint8_t *>(st + 8 * M);                         // [M][kQRow]
    __shared__ uint32_t phase_s[kBufs][4], top_s[kSets][4];

    // Row tiles of one (KV head, run) follow each other on one XCD (workgroups go round the eight of them), so that they find its
    // blocks in that L2.
    const uint32_t groups = (uint32_t)p.BH * (uint32_t)p.nsplit, seq = blockIdx.x >> 3;
    const uint32_t group = (seq / (uint32_t)p.row_tiles) * 8u + (blockIdx.x & 7u);
    if (group >= groups) return;
    const int rt = (int)(seq % (uint32_t)p.row_tiles), bh = (int)(group % (uint32_t)p.BH), split = (int)(group / (uint32_t)p.BH);
    const int b = bh / p.Hkv, hkv = bh % p.Hkv;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, t = lane & 31;
    const int tr = R16 ? lane & 15 : t, g = lane >> 4;     // this lane's row of a block; sixteen rows: its quarter of what the products add up
    const int rg = wave >> 2, quarter = wave & 3;          // rows, and tokens, of this wavefront
    const int T = p.T_c + p.T_w;
    const int row0 = rt * M, row_last = min(row0 + M, p.rows) - 1, mine0 = 32 * NB * rg;
    const int start = p.starts ? min(max(p.starts[b], 0), T) : 0;
    const int pos_first = p.causal ? T - p.n + min(row0 + mine0, p.rows - 1) / p.G : T - 1, pos_last = p.causal ? T - p.n + row_last / p.G : T - 1;

    int row[NB], pos[NB];                                  // the lane's rows, and the last token that each sees
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        row[nb] = min(row0 + mine0 + 32 * nb + tr, p.rows - 1);
        pos[nb] = p.causal ? T - p.n + row[nb] / p.G : T - 1;
    }
    auto q_row = [&](int r) -> const uint16_t * {
        return p.q + (int64_t)b * p.q_b + (int64_t)(hkv * p.G + r % p.G) * p.q_h + (int64_t)(r / p.G) * p.q_t;
    };

    // ---- this run's tiles: compressed ones [c0, c1), then window ones [w0, w1) ----
    const int first = split * p.run, last = min(first + p.run, p.tiles);
    const int seen_c = min(p.T_c, pos_last + 1);           // (tokens behind the last row's own are nobody's)
    const int c0 = max(first, start / kChunkTile), c1 = min(last, (seen_c + kChunkTile - 1) / kChunkTile);
    const int w0 = max(first - p.tiles_c, max(start - p.T_c, 0) / kChunkTile), w1 = min(last - p.tiles_c, (pos_last - p.T_c) / kChunkTile + 1);

    // ---- staging of a tile's four blocks (quarter = block), ahead of their use; block_info a tile further, through scalar loads ----
    typedef const __attribute__((address_space(4))) uint32_t *const_u32_ptr;
    const uint32_t cap = quarter < 2 ? (uint32_t)k_block_bound(64, p.k_bits) : (uint32_t)v_block_bound(64, p.v_bits);
    const uint64_t bytes = quarter < 2 ? p.k_bytes : p.v_bytes;
    const const_u32_ptr info = reinterpret_cast<const_u32_ptr>(reinterpret_cast<uintptr_t>(quarter < 2 ? p.k_info : p.v_info));
    const uint32_t blk0 = quarter < 2 ? (uint32_t)quarter * (uint32_t)p.BH + (uint32_t)bh : 2u * (uint32_t)bh + (uint32_t)(quarter - 2);
    uint32_t next_off = 0, next_size = 0;
    auto look_up = [&](int tile) {
        const size_t at = 2 * ((size_t)blk0 + 2 * (size_t)min(tile, p.tiles_c - 1) * (size_t)p.BH);
        next_off = info[at];
        next_size = info[at + 1];
    };
    const uint32_t bytes4 = (uint32_t)((bytes + 3u) & ~3ull);
    const uintptr_t stream = reinterpret_cast<uintptr_t>(quarter < 2 ? p.k_stream : p.v_stream);
    const u4 copy_rsrc = {(uint32_t)stream, (uint32_t)(stream >> 32) & 0xFFFFu, bytes4, 0x00020000u};
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(stream), 0, (int)bytes4, 0x00020000);
    const uint32_t slot = quarter < 2 ? p.slot_k : p.slot_v;
    auto block_at = [&](int side, int j, int tile_nr) -> uint32_t {            // tile_nr: counted from the run's first
        return side ? 2u * kKBufs * p.slot_k + (uint32_t)(2 * (tile_nr % kBufs) + j) * p.slot_v : (uint32_t)(2 * (tile_nr % kKBufs) + j) * p.slot_k;
    };
    u4 raw[COPY ? 1 : NQ];
    uint32_t raw_phase = 0, par_k = 0, par_kz = 0, par_v = 0, par_vz = 0;
    // starts the copies of `tile`, whose entry look_up has fetched (COPY = false: into registers, for put)
    auto fetch = [&](int tile) {
        uint32_t off = next_off, size = min(next_size, cap);               // (never outside the stream, whatever block_info says)
        if ((uint64_t)off > bytes) off = (uint32_t)bytes;
        size = (uint32_t)min((uint64_t)size, bytes - (uint64_t)off);
        raw_phase = off & 15u;
        const uint32_t n16 = (raw_phase + size + 15u) >> 4, src = off - raw_phase;
        if (!COPY) {
#pragma unroll
            for (int i = 0; i < (COPY ? 1 : NQ); i++) {
                const uint32_t c = (uint32_t)(lane + 64 * i);
                raw[i] = c < n16 ? __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, src + 16u * c, 0, 0)) : (u4){0, 0, 0, 0};
            }
        } else {
            const uint32_t dst = (uint32_t)reinterpret_cast<uintptr_t>(ring) + block_at(quarter >> 1, quarter & 1, tile - c0);
#pragma unroll
            for (int i = 0; i < (NQ + RG - 1) / RG; i++) {                 // (two groups of rows: every other step each)
                const uint32_t step = (uint32_t)(RG * i + rg);
                if ((uint32_t)lane + 64u * step < n16) copy_to_lds(copy_rsrc, __builtin_amdgcn_readfirstlane(dst + 1024u * step), src + 16u * ((uint32_t)lane + 64u * step));
            }
            if (lane == 0 && rg == 0) phase_s[(tile - c0) % kBufs][quarter] = raw_phase;
        }
        look_up(tile + 1);
    };
    auto fetch_par = [&](int tile) {                       // the parameters of this wavefront's 32 tokens
        const size_t at = (size_t)b * p.par_stride + (size_t)tile * kChunkTile + 32 * quarter + t;
        par_k = p.k_scale[at]; par_kz = p.k_zero[at]; par_v = p.v_scale[at]; par_vz = p.v_zero[at];
    };
    auto put = [&](int tile) {                             // what fetch has started is in LDS behind the next barrier
        if (!COPY) {
            uint8_t *dst = ring + block_at(quarter >> 1, quarter & 1, tile - c0);
#pragma unroll
            for (int i = 0; i < (COPY ? 1 : NQ); i++)
                if ((uint32_t)(lane + 64 * i) * 16u < slot) *reinterpret_cast<u4 *>(dst + 16 * (lane + 64 * i)) = raw[i];
            if (lane == 0) phase_s[(tile - c0) % kBufs][quarter] = raw_phase;
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
    };
    if (c0 < c1) {
        look_up(c0);
        if (!ONCE || quarter < 2) fetch(c0);
        if (RG == 2 && c0 + 1 < c1) fetch(c0 + 1);
        fetch_par(c0);
    }

    // ---- q: rows into LDS as fp16 (bf16: times 2^up), their sums ----
    constexpr int kPieces = M * 16 / (256 * RG);           // of 16 bytes, a thread
    u4 qw[kPieces];
#pragma unroll
    for (int j = 0; j < kPieces; j++) {
        const int i = tid + 256 * RG * j;
        qw[j] = *reinterpret_cast<const u4 *>(q_row(min(row0 + (i >> 4), p.rows - 1)) + 8 * (i & 15));
    }
    int up = 0;
    bool apart = false;                                    // rows further apart than 2^8: each has a power of two of its own on top
    if (BF) {
        typedef unsigned short u16pair __attribute__((ext_vector_type(2)));
        uint32_t high[kPieces];                            // a row's largest size; 0: it sees nothing, or holds nothing finite but zeroes
        u16pair both = {0, 0};                             // the largest of the rows', 0x7FFF - the least
#pragma unroll
        for (int j = 0; j < kPieces; j++) {                // (infinities, NaN and rows that see nothing do not count)
            const int r = min(row0 + ((tid + 256 * RG * j) >> 4), p.rows - 1);
            uint32_t most = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t lo = qw[j][k] & 0x7FFFu, hi = (qw[j][k] >> 16) & 0x7FFFu;
                most = max(most, max(lo < 0x7F80u ? lo : 0u, hi < 0x7F80u ? hi : 0u));
            }
            most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0xB1, 0xF, 0xF, true));   // (sixteen lanes a row: pairs,
            most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0x4E, 0xF, 0xF, true));   // fours,
            most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0x141, 0xF, 0xF, true));  // eights mirrored,
            most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0x140, 0xF, 0xF, true));  // sixteens mirrored)
            high[j] = !p.causal || T - p.n + r / p.G >= start ? most : 0u;
            both = __builtin_elementwise_max(both, (u16pair){(unsigned short)high[j], (unsigned short)(high[j] ? 0x7FFFu - high[j] : 0u)});
        }
#pragma unroll
        for (int d = 32; d >= 16; d >>= 1)
            both = __builtin_elementwise_max(both, __builtin_bit_cast(u16pair, __shfl_xor(__builtin_bit_cast(int, both), d, 64)));
        if (lane == 0) tab_all[wave] = __builtin_bit_cast(uint32_t, both);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4 * RG; i++) both = __builtin_elementwise_max(both, __builtin_bit_cast(u16pair, tab_all[i]));
        const uint32_t top = both[0], least = 0x7FFFu - both[1];
        up = top ? min(max(141 - (int)(top >> 7), -120), 120) : 0;        // the largest comes to 2^14 .. 2^15
        apart = __builtin_amdgcn_readfirstlane((int)(top >> 7) - (int)(least >> 7)) >= 8;
#pragma unroll
        for (int j = 0; j < kPieces; j++) {
            const int i = tid + 256 * RG * j, own = apart && high[j] ? min((int)(top >> 7) - (int)(high[j] >> 7), 100 - max(up - 20, 0)) : 0;
            const float up_f = __uint_as_float((uint32_t)(127 + up + own) << 23);
#pragma unroll
            for (int k = 0; k < 4; k++) qw[j][k] = pack_f16(__uint_as_float(qw[j][k] << 16) * up_f, __uint_as_float(qw[j][k] & 0xFFFF0000u) * up_f);
            if ((i & 15) == 0) st[i >> 4] = __uint_as_float((uint32_t)(127 - own) << 23);      // (scores are taken times that; the place is the end's)
        }
    }
#pragma unroll
    for (int j = 0; j < kPieces; j++) {
        const int i = tid + 256 * RG * j;
        *reinterpret_cast<u4 *>(qt + (i >> 4) * kQRow + 16 * (i & 15)) = qw[j];
    }
    if (c0 < c1) put(c0);
    __syncthreads();
    float qsum[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {                      // half the channels each (a quarter)
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < (R16 ? 4 : 8); c++) {
            const h8 v = *reinterpret_cast<const h8 *>(qt + (mine0 + 32 * nb + tr) * kQRow + (R16 ? 64 * c + 16 * g : 32 * c + 16 * h));
#pragma unroll
            for (int k = 0; k < 8; k++) s += (float)v[k];
        }
        if (R16) s += __shfl_xor(s, 16, 64);
        qsum[nb] = s + __shfl_xor(s, 32, 64);
        if (BF && apart) qsum[nb] *= st[mine0 + 32 * nb + tr];
    }

    f16v acc[NB][4];
    f4v acc16[8];
    float m[NB], l[NB], z[NB];
#pragma unroll
    for (int c = 0; c < 8; c++) acc16[c] = (f4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        m[nb] = kLowest; l[nb] = 0.f; z[nb] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[nb][c][r] = 0.f;
    }
    const float to_score = p.sm_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
    uint32_t emax = 0;                                     // exponent field of the largest V scale met, at least 14; 0: none yet
    float unit = 1.f;                                      // result = (acc + z) * unit
    const UnitGeom gk = unit_geom(p.k_bits), gv = unit_geom(p.v_bits);
    if (!WIDE) { __builtin_assume(gk.W <= 4); __builtin_assume(gv.W <= 4); }
    const int tau = (t & 3) + 4 * (t >> 3) + 16 * ((t >> 2) & 1);          // the token (of 32) in row t of S^T: lane half = pack

    // A half-wavefront's unit of a staged tile: where it starts in its block.
    const int hw = 2 * quarter + h, u = hw & 3;
    auto unit_start = [&](int tile, int side, uint32_t blk_at) -> uint32_t {
        const uint32_t phase = phase_s[(tile - c0) % kBufs][2 * side + (hw >> 2)];
        const uint8_t *blk = ring + blk_at;
        return min(phase + 8u + (u ? (uint32_t)reinterpret_cast<const uint16_t *>(blk + phase)[u - 1] : 0u), (side ? p.slot_v : p.slot_k) - 16u);
    };
    auto unpack_k = [&](int tile, uint8_t *kt) {           // 16 tokens x 128 channels; the quarter's two units make its 32 tokens
        uint8_t *dst = kt + quarter * 32 * kKRow + 16 * h * kKRow + 4 * t;
        const uint32_t blk_at = block_at(0, hw >> 2, tile - c0);
        const uint32_t at = unit_start(tile, 0, blk_at);
        const auto put_codes = [&](int k, uint32_t c4) { *reinterpret_cast<uint32_t *>(dst + k * kKRow) = c4; };
        if (WIDE) {
            unit_codes(ring + blk_at, at, t, gk, put_codes);
        } else {
            UnitPacks packs;
            uint32_t where[4];
            narrow_packs(ring + blk_at + at, t, gk, packs.len, packs.mn, where);
#pragma unroll
            for (int i = 0; i < 4; i++) packs.word[i] = lds_load64(ring, blk_at + at + where[i]);
            packs_codes(packs, put_codes);
        }
    };
    auto parse_v = [&](int tile, uint32_t *tab) {          // where the unit's packs are
        const uint32_t blk_at = block_at(1, hw >> 2, tile - c0), at = unit_start(tile, 1, blk_at);
        const uint8_t *blk = ring + blk_at;
        if (!WIDE) {                                       // (damaged fields reach 2 KiB behind what is staged, at K's codes)
            uint32_t len[4], mn[4], where[4];
            narrow_packs(blk + at, t, gv, len, mn, where);
#pragma unroll
            for (int i = 0; i < 4; i++) tab[(hw * 4 + i) * 32 + t] = (blk_at + at + where[i]) | (len[i] << 17) | (mn[i] << 21);
            return;
        }
        const uint32_t minsw = lds_meta_word(blk + at, t, gv.W), lensw = lds_meta_word(blk + at + gv.mins_bytes, t, gv.LB);
        uint32_t len[4], off[4], payload;
#pragma unroll
        for (int i = 0; i < 4; i++) len[i] = min((lensw >> (i * gv.LB)) & ((1u << gv.LB) - 1u), (uint32_t)gv.W);
        pack_offsets(len, off, payload);
        const uint32_t base = blk_at + at + (uint32_t)(gv.mins_bytes + gv.lens_bytes);
#pragma unroll
        for (int i = 0; i < 4; i++)
            tab[(hw * 4 + i) * 32 + t] = min(base + off[i], p.ring - 32u) | (len[i] << 17) | (((minsw >> (i * gv.W)) & ((1u << gv.W) - 1u)) << 21);
    };
    // Parameters of the quarter's 32 tokens into LDS; those in front of the sequence count as nothing.  Returns what the accumulators
    // are to be multiplied with where a larger V scale than before came up.  (Two groups of rows: the group that writes and the one
    // that reads follow the same scales.)
    auto raise_scale = [&](uint32_t e) -> float {
        float grow = 1.f;
        if (e > emax) {
            if (emax) grow = __builtin_amdgcn_exp2f((float)(int)(emax - e));
            emax = e;
            unit = __uint_as_float((e - 6u) << 23);        // 1 / (the weights' power of two, 2^(133 - e): V scales come to 2^7 at most)
        }
        return grow;
    };
    uint32_t writer_top = 0;                               // the largest V scale that the parameters in LDS have met
    auto write_par = [&](int tile, int set) -> uint32_t {
        const bool real = tile * kChunkTile + 32 * quarter + t >= start;
        const float ks = real ? chunk_f32(par_k, BF) * to_score : 0.f, kz = real ? chunk_f32(par_kz, BF) : 0.f;
        const float vs = real ? chunk_f32(par_v, BF) : 0.f, vz = real ? chunk_f32(par_vz, BF) : 0.f;
        const uint32_t e = max(half_max((__float_as_uint(vs) >> 23) & 255u), 14u);
        writer_top = max(writer_top, e);
        const float vw = vs * __uint_as_float((260u - writer_top) << 23);
        float2 *dst = par_all + set * 256 + quarter * 32 + t;
        if (h == 0) {
            dst[0] = make_float2(ks, kz * ks);
            dst[128] = make_float2(vw, vz);
        }
        return e;
    };

    // Scores of a tile's 32 tokens against the lane's rows, the softmax step, and the weights as operands.
    auto weights_of = [&](int tile, const uint8_t *kt, const float2 *par, float grow, u4 (&w)[NB][2]) {
        const int tok0 = tile * kChunkTile + 32 * quarter;                     // this wavefront's first token
        kt += quarter * 32 * kKRow;
        const float2 *par_s = par + quarter * 32, *par_w = par_s + 128;
        f16v y[NB];
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int r = 0; r < 16; r++) y[nb][r] = 0.f;
#pragma unroll
        for (int s = 0; s < 8; s++) {
            const uint2 c8 = *reinterpret_cast<const uint2 *>(kt + tau * kKRow + 16 * s + 8 * h);
            const u4 a = {codes_f16(c8.x, 0x04010400u), codes_f16(c8.x, 0x04030402u), codes_f16(c8.y, 0x04010400u), codes_f16(c8.y, 0x04030402u)};
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
                y[nb] = product<false>(a, *reinterpret_cast<const u4 *>(qt + (mine0 + 32 * nb + t) * kQRow + 32 * s + 16 * h), y[nb]);
        }
        if (BF && apart) {
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                const float down = st[mine0 + 32 * nb + t];
#pragma unroll
                for (int r = 0; r < 16; r++) y[nb][r] *= down;
            }
        }
        float ref[NB];                                     // what the scores are taken against
#pragma unroll
        for (int nb = 0; nb < NB; nb++) ref[nb] = m[nb] == kLowest ? 0.f : m[nb];
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const float2 q2 = par_s[16 * h + r];
#pragma unroll
            for (int nb = 0; nb < NB; nb++) y[nb][r] = fmaf(y[nb][r], q2.x, fmaf(q2.y, qsum[nb], -ref[nb]));
        }
        if (tok0 + 31 > pos_first || tok0 < start) {       // (uniform: some row does not see every token)
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                int up_to = pos[nb] - (tok0 + 16 * h), from = start - (tok0 + 16 * h);
                asm volatile("" : "+v"(up_to), "+v"(from));                    // (a branch, not a hundred selects that every tile pays for)
#pragma unroll
                for (int r = 0; r < 16; r++) y[nb][r] = r > up_to || r < from ? -INFINITY : y[nb][r];
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            float over = y[nb][0];
#pragma unroll
            for (int r = 1; r < 16; r++) over = fmaxf(over, y[nb][r]);
            if (__any(over > 8.f || m[nb] == kLowest) || grow != 1.f || tok0 + 31 > pos_first) {
                over = fmaxf(over, __shfl_xor(over, 32, 64));
                const bool none = m[nb] == kLowest, some = over > -INFINITY;
                float raise = over > 8.f || (none && some) ? over : 0.f;
                if (tok0 + 31 > pos_first) {               // (tokens that some row does not see: never for most tiles)
                    float most = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; r++) most = fmaxf(most, y[nb][r] > -INFINITY ? fabsf(par_w[16 * h + r].x) : 0.f);
                    most = fmaxf(most, __shfl_xor(most, 32, 64));
                    const float sum = l[nb] + __shfl_xor(l[nb], 32, 64);
                    raise -= unseen_shift(most, sum > 0.f ? 64.f * grow : 0.f, sum);
                }
                if (!none || some) m[nb] = ref[nb] + raise;
                const float alpha = none ? 1.f : __builtin_amdgcn_exp2f(-raise);           // (nothing is summed before the first)
#pragma unroll
                for (int r = 0; r < 16; r++) y[nb][r] -= raise;
                l[nb] *= alpha;
                z[nb] *= alpha * grow;
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[nb][c][r] *= alpha * grow;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float2 pa = par_w[16 * h + j], pb = par_w[16 * h + j + 8];
                const float a = __builtin_amdgcn_exp2f(y[nb][j]), d = __builtin_amdgcn_exp2f(y[nb][j + 8]);
                l[nb] += a;
                l[nb] += d;
                uint32_t f = pack_f16(a * pa.x, d * pb.x);
                asm("" : "+v"(f));                         // (the sum takes these very halves: formed again they round once less)
                const h2v f2 = __builtin_bit_cast(h2v, f);
                z[nb] = fmaf((float)f2[0], pa.y, z[nb]);
                z[nb] = fmaf((float)f2[1], pb.y, z[nb]);
                w[nb][j >> 2][j & 3] = f;
            }
        }
    };
    auto add_values = [&](const uint32_t *tab, const u4 (&w)[NB][2]) {
#pragma unroll
        for (int c = 0; c < 4; c++) {                      // 32 channels: block c / 2, column of units c % 2
            const uint32_t e = tab[((((c >> 1) * 4 + (c & 1) * 2 + (quarter >> 1)) * 4) + 2 * (quarter & 1) + h) * 32 + t];
            uint32_t v[8];
            pack_operand<WIDE>(ring, e, v);
            const u4 v0 = {v[0], v[1], v[2], v[3]}, v1 = {v[4], v[5], v[6], v[7]};
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                acc[nb][c] = product<false>(v0, w[nb][0], acc[nb][c]);
                acc[nb][c] = product<false>(v1, w[nb][1], acc[nb][c]);
            }
        }
    };

    // Sixteen rows (R16): the same on 16x16x32 products, which leave no columns idle.  S^T's two products are tokens 0..7 and 8..15 of
    // either pack, so that a lane's scores of the two are the pairs (j, j + 8) of an operand: packs g / 2, tokens 4 (g % 2) + i and that + 8.
    // V is unpacked as above, a pack a lane; its halves change places between neighbouring rows of 16 lanes, which makes of 32 channels'
    // packs the operands of 16 and 16.
    const int base16 = 16 * (g >> 1) + 4 * (g & 1), tok16 = 16 * ((lane & 15) >> 3) + (lane & 7);
    auto weights_of_16 = [&](int tile, const uint8_t *kt, const float2 *par, float grow, u4 &w) {
        const int tok0 = tile * kChunkTile + 32 * quarter;
        kt += quarter * 32 * kKRow;
        const float2 *par_s = par + quarter * 32 + base16, *par_w = par_s + 128;
        f4v y[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const u4 b = *reinterpret_cast<const u4 *>(qt + tr * kQRow + 64 * s + 16 * g);
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const uint2 c8 = *reinterpret_cast<const uint2 *>(kt + (tok16 + 8 * n) * kKRow + 32 * s + 8 * g);
                const u4 a = {codes_f16(c8.x, 0x04010400u), codes_f16(c8.x, 0x04030402u), codes_f16(c8.y, 0x04010400u), codes_f16(c8.y, 0x04030402u)};
                y[n] = product16<false>(a, b, y[n]);
            }
        }
        if (BF && apart) {
            const float down = st[tr];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i >> 2][i & 3] *= down;
        }
        const float ref = m[0] == kLowest ? 0.f : m[0];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 q2 = par_s[8 * n + i];
                y[n][i] = fmaf(y[n][i], q2.x, fmaf(q2.y, qsum[0], -ref));
            }
        if (tok0 + 31 > pos_first || tok0 < start) {
            int up_to = pos[0] - (tok0 + base16), from = start - (tok0 + base16);
            asm volatile("" : "+v"(up_to), "+v"(from));
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) y[n][i] = 8 * n + i > up_to || 8 * n + i < from ? -INFINITY : y[n][i];
        }
        float over = y[0][0];
#pragma unroll
        for (int i = 1; i < 8; i++) over = fmaxf(over, y[i >> 2][i & 3]);
        if (__any(over > 8.f || m[0] == kLowest) || grow != 1.f || tok0 + 31 > pos_first) {
            over = fmaxf(over, __shfl_xor(over, 16, 64));
            over = fmaxf(over, __shfl_xor(over, 32, 64));
            const bool none = m[0] == kLowest, some = over > -INFINITY;
            float raise = over > 8.f || (none && some) ? over : 0.f;
            if (tok0 + 31 > pos_first) {
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) most = fmaxf(most, y[i >> 2][i & 3] > -INFINITY ? fabsf(par_w[8 * (i >> 2) + (i & 3)].x) : 0.f);
                most = fmaxf(most, __shfl_xor(most, 16, 64));
                most = fmaxf(most, __shfl_xor(most, 32, 64));
                float sum = l[0] + __shfl_xor(l[0], 16, 64);
                sum += __shfl_xor(sum, 32, 64);
                raise -= unseen_shift(most, sum > 0.f ? 64.f * grow : 0.f, sum);
            }
            if (!none || some) m[0] = ref + raise;
            const float alpha = none ? 1.f : __builtin_amdgcn_exp2f(-raise);
#pragma unroll
            for (int i = 0; i < 8; i++) y[i >> 2][i & 3] -= raise;
            l[0] *= alpha;
            z[0] *= alpha * grow;
#pragma unroll
            for (int c = 0; c < 8; c++) acc16[c] *= alpha * grow;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 pa = par_w[i], pb = par_w[i + 8];
            const float a = __builtin_amdgcn_exp2f(y[0][i]), d = __builtin_amdgcn_exp2f(y[1][i]);
            l[0] += a;
            l[0] += d;
            uint32_t f = pack_f16(a * pa.x, d * pb.x);
            asm("" : "+v"(f));
            const h2v f2 = __builtin_bit_cast(h2v, f);
            z[0] = fmaf((float)f2[0], pa.y, z[0]);
            z[0] = fmaf((float)f2[1], pb.y, z[0]);
            w[i] = f;
        }
    };
    auto add_values_16 = [&](const uint32_t *tab, const u4 &w) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint32_t e = tab[((((c >> 1) * 4 + (c & 1) * 2 + (quarter >> 1)) * 4) + 2 * (quarter & 1) + h) * 32 + t];
            uint32_t v[8];
            pack_operand<false>(ring, e, v);
            u4 lo, hi;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const auto both = __builtin_amdgcn_permlane16_swap(v[i], v[4 + i], false, false);
                lo[i] = both[0];
                hi[i] = both[1];
            }
            acc16[2 * c] = product16<false>(lo, w, acc16[2 * c]);
            acc16[2 * c + 1] = product16<false>(hi, w, acc16[2 * c + 1]);
        }
    };

    // ---- compressed tiles ----
    const auto lds_barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };      // (copies go on)
    if (ONCE) {
        // Few rows: three workgroups a CU cover each other's waits, with one place for K's blocks and one for V's: V's are copied while the
        // scores are formed, the next tile's K during the products with V.  Three barriers a tile: K, V, table.
        for (int tile = c0; tile < c1; tile++) {
            if (tile != c0) {
                put(tile);
                lds_barrier();                             // (and the table's readers are done)
            }
            if (quarter >= 2) fetch(tile);
            const float grow = raise_scale(write_par(tile, 0));
            unpack_k(tile, kt_all);
            wave_lds_order();
            u4 w[NB][2];
            if constexpr (R16) weights_of_16(tile, kt_all, par_all, grow, w[0][0]);
            else weights_of(tile, kt_all, par_all, grow, w);
            put(tile);
            lds_barrier();
            if (tile + 1 < c1) {
                if (quarter < 2) fetch(tile + 1);
                fetch_par(tile + 1);
            }
            parse_v(tile, tab_all);
            lds_barrier();
            if constexpr (R16) add_values_16(tab_all, w[0][0]);
            else add_values(tab_all, w);
        }
    } else if (RG == 1) {
        // Few rows and wide codes: two workgroups a CU cover each other's waits.  Two barriers a tile: staged blocks, table.
        for (int tile = c0; tile < c1; tile++) {
            if (tile != c0) __syncthreads();               // the tile is staged, and the table's readers are done
            const float grow = raise_scale(write_par(tile, 0));
            if (tile + 1 < c1) {
                fetch(tile + 1);
                fetch_par(tile + 1);
            }
            parse_v(tile, tab_all);
            unpack_k(tile, kt_all);
            wave_lds_order();
            u4 w[NB][2];
            weights_of(tile, kt_all, par_all, grow, w);
            __syncthreads();
            add_values(tab_all, w);
            if (tile + 1 < c1) put(tile + 1);
        }
    } else if (c0 < c1) {
        // Many rows: the two groups of rows share what is unpacked -- the first group's wavefronts unpack K, the second's find V's
        // packs and write the parameters, a tile ahead, while the others are at their products.  One barrier a tile.
        auto prepare = [&](int tile, int set) {
            if (rg == 0) {
                unpack_k(tile, kt_all + set * 4 * 32 * kKRow);
            } else {
                parse_v(tile, tab_all + set * 1024);
                const uint32_t e = write_par(tile, set);
                if (lane == 0) top_s[set][quarter] = e;
            }
        };
        prepare(c0, 0);
        if (rg == 1 && c0 + 1 < c1) fetch_par(c0 + 1);
        __syncthreads();
        for (int tile = c0; tile < c1; tile++) {
            const int set = (tile - c0) & 1;
            if (tile + 2 < c1) fetch(tile + 2);
            if (tile + 1 < c1) {
                prepare(tile + 1, set ^ 1);
                if (rg == 1 && tile + 2 < c1) fetch_par(tile + 2);
            }
            const float grow = raise_scale(__builtin_amdgcn_readfirstlane(top_s[set][quarter]));
            u4 w[NB][2];
            weights_of(tile, kt_all + set * 4 * 32 * kKRow, par_all + set * 256, grow, w);
            add_values(tab_all + set * 1024, w);
            put(tile + 2);
            __syncthreads();
        }
    }

    // What the rest needs of the arguments is read again here: held in scalar registers across the loop above it made that loop spill.
    typedef const __attribute__((address_space(4))) ChunkParams *late_ptr;
    late_ptr late = reinterpret_cast<late_ptr>(reinterpret_cast<uintptr_t>(__builtin_amdgcn_kernarg_segment_ptr()));
    asm volatile("" : "+s"(late));

    // ---- window tiles: the same products on the 16-bit rows ----
    if (w0 < w1) {
        __syncthreads();                                   // the staged blocks are dead
        constexpr float kUp = BF ? 1.f : 16384.f;          // fp16 weights: 2^14 p, so that small ones keep their bits
        if (emax) {
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                z[nb] = z[nb] * unit * kUp;
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[nb][c][r] = acc[nb][c][r] * unit * kUp;
            }
#pragma unroll
            for (int c = 0; c < 8; c++) acc16[c] = acc16[c] * unit * kUp;
        }
        unit = 1.f / kUp;
        uint8_t *vt = ring + wave * 32 * kVRow;            // (into the K codes' place, where two groups of rows need it)
        for (int wt = w0; wt < w1; wt++) {
            const int r0 = wt * kChunkTile + 32 * quarter, tok0 = late->T_c + r0;     // window row and position of the wavefront's first token
            if (r0 >= late->T_w || tok0 > pos_last || tok0 + 31 < start) continue; // (uniform, and no barrier in here)
            const uint16_t *kr = late->k_win + ((size_t)bh * late->win_stride + min(r0 + tau, late->T_w - 1)) * kHeadDim + 8 * h;
            const uint16_t *vr = late->v_win + ((size_t)bh * late->win_stride) * kHeadDim;
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < 8; i++) {                  // four rows of V a step, 16 lanes each; rows that nobody sees as zeroes
                const int k = 4 * i + (lane >> 4), c = lane & 15;
                const bool real = r0 + k < late->T_w && tok0 + k >= start && tok0 + k <= pos_last;
                const uint2 *src = reinterpret_cast<const uint2 *>(vr + (size_t)min(r0 + k, late->T_w - 1) * kHeadDim + 8 * c);
                const uint2 a = src[0], d = src[1];
                uint2 *dst = reinterpret_cast<uint2 *>(vt + k * kVRow + 16 * c);
                dst[0] = real ? a : make_uint2(0u, 0u);
                dst[1] = real ? d : make_uint2(0u, 0u);
            }
            if constexpr (R16) {
                f4v y[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
                const uint16_t *kw = late->k_win + (size_t)bh * late->win_stride * kHeadDim + 8 * g;
                const uint16_t *qr = late->q + (int64_t)b * late->q_b + (int64_t)(hkv * late->G + row[0] % late->G) * late->q_h + (int64_t)(row[0] / late->G) * late->q_t;
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const u4 x = BF ? *reinterpret_cast<const u4 *>(qr + 32 * s + 8 * g) : *reinterpret_cast<const u4 *>(qt + tr * kQRow + 64 * s + 16 * g);
#pragma unroll
                    for (int n = 0; n < 2; n++)
                        y[n] = product16<BF>(*reinterpret_cast<const u4 *>(kw + (size_t)min(r0 + tok16 + 8 * n, late->T_w - 1) * kHeadDim + 32 * s), x, y[n]);
                }
                float most = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int tok = tok0 + base16 + 8 * (i >> 2) + (i & 3);
                    const float x = tok > pos[0] || tok < start ? -INFINITY : y[i >> 2][i & 3] * late->sm_log2;
                    y[i >> 2][i & 3] = x;
                    most = fmaxf(most, x);
                }
                most = fmaxf(most, __shfl_xor(most, 16, 64));
                most = fmaxf(most, __shfl_xor(most, 32, 64));
                const float was = m[0];
                m[0] = fmaxf(was, most);
                const float alpha = __builtin_amdgcn_exp2f(was - m[0]);
                l[0] *= alpha;
                z[0] *= alpha;
#pragma unroll
                for (int c = 0; c < 8; c++) acc16[c] *= alpha;
                u4 w, wl;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float a = __builtin_amdgcn_exp2f(y[0][i] - m[0]), d = __builtin_amdgcn_exp2f(y[1][i] - m[0]);
                    l[0] += a + d;
                    w[i] = BF ? pack_bf16(a, d) : pack_f16(a * kUp, d * kUp);
                    wl[i] = BF ? pack_bf16(a - __uint_as_float(w[i] << 16), d - __uint_as_float(w[i] & 0xFFFF0000u)) : 0u;
                }
                wave_lds_order();
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const uint16_t *col = reinterpret_cast<const uint16_t *>(vt + base16 * kVRow) + 16 * c + (lane & 15);
                    u4 v;
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = (uint32_t)col[i * (kVRow / 2)] | ((uint32_t)col[(i + 8) * (kVRow / 2)] << 16);
                    acc16[c] = product16<BF>(v, w, acc16[c]);
                    if (BF) acc16[c] = product16<BF>(v, wl, acc16[c]);
                }
                continue;
            }
            f16v y[NB];
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int r = 0; r < 16; r++) y[nb][r] = 0.f;
#pragma unroll
            for (int s = 0; s < 8; s++) {
                const u4 a = *reinterpret_cast<const u4 *>(kr + 16 * s);
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
                    y[nb] = product<BF>(a, BF ? *reinterpret_cast<const u4 *>((late->q + (int64_t)b * late->q_b + (int64_t)(hkv * late->G + row[nb] % late->G) * late->q_h + (int64_t)(row[nb] / late->G) * late->q_t) + 16 * s + 8 * h)
                                              : *reinterpret_cast<const u4 *>(qt + (mine0 + 32 * nb + t) * kQRow + 32 * s + 16 * h), y[nb]);
            }
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int tok = tok0 + 16 * h + r;
#pragma unroll
                for (int nb = 0; nb < NB; nb++) y[nb][r] = tok > pos[nb] || tok < start ? -INFINITY : y[nb][r] * late->sm_log2;
            }
            wave_lds_order();
            u4 w[NB][2], wl[NB][2];                        // bf16: what the rounding leaves goes through the matrix cores as well
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                const float alpha = softmax_step(y[nb], m[nb]);
                l[nb] *= alpha;
                z[nb] *= alpha;
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[nb][c][r] *= alpha;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float a = y[nb][j], d = y[nb][j + 8];
                    l[nb] += a + d;
                    if (BF) {
                        const uint32_t hi = pack_bf16(a, d);
                        w[nb][j >> 2][j & 3] = hi;
                        wl[nb][j >> 2][j & 3] = pack_bf16(a - __uint_as_float(hi << 16), d - __uint_as_float(hi & 0xFFFF0000u));
                    } else {
                        w[nb][j >> 2][j & 3] = pack_f16(a * kUp, d * kUp);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint16_t *col = reinterpret_cast<const uint16_t *>(vt + 16 * h * kVRow) + 32 * c + t;
                u4 v[2];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j >> 2][j & 3] = (uint32_t)col[j * (kVRow / 2)] | ((uint32_t)col[(j + 8) * (kVRow / 2)] << 16);
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        acc[nb][c] = product<BF>(v[e], w[nb][e], acc[nb][c]);
                        if (BF) acc[nb][c] = product<BF>(v[e], wl[nb][e], acc[nb][c]);
                    }
            }
        }
    }

    // ---- the states of a row's four wavefronts become one ----
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        if (R16) {
            l[nb] += __shfl_xor(l[nb], 16, 64);
            z[nb] += __shfl_xor(z[nb], 16, 64);
        }
        l[nb] += __shfl_xor(l[nb], 32, 64);
        z[nb] += __shfl_xor(z[nb], 32, 64);
        if (R16 ? g == 0 : h == 0) st[quarter * M + mine0 + 32 * nb + tr] = m[nb];
    }
    __syncthreads();
    float *sums = st + 4 * M;
    float top[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const float *at = st + mine0 + 32 * nb + tr;
        top[nb] = fmaxf(fmaxf(at[0], at[M]), fmaxf(at[2 * M], at[3 * M]));
        const float f = __builtin_amdgcn_exp2f(m[nb] - top[nb]);
        if (R16 ? g == 0 : h == 0) sums[quarter * M + mine0 + 32 * nb + tr] = l[nb] * f;
        const float fu = f * unit;
#pragma unroll
        for (int c = 0; c < 8; c++) acc16[c] = (acc16[c] + z[nb]) * fu;
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[nb][c][r] = (acc[nb][c][r] + z[nb]) * fu;
    }
    constexpr int kSumRow = 129;
    float *buf0 = reinterpret_cast<float *>(ring) + rg * 2 * 32 * kSumRow;           // [2][32 rows][129]: quarters 0 + 2 and 1 + 3
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        float *mine = buf0 + (quarter & 1) * 32 * kSumRow + t * kSumRow + 4 * h;
#pragma unroll
        for (int step = 0; step < 2; step++) {
            if ((quarter >> 1) == step && R16) {
#pragma unroll
                for (int c = 0; c < 8; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float *at = buf0 + (quarter & 1) * 32 * kSumRow + tr * kSumRow + 16 * c + 4 * g + i;
                        *at = step ? *at + acc16[c][i] : acc16[c][i];
                    }
            } else if ((quarter >> 1) == step) {
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        float *at = mine + 32 * c + 8 * (r >> 2) + (r & 3);
                        *at = step ? *at + acc[nb][c][r] : acc[nb][c][r];
                    }
            }
            __syncthreads();
        }
        const int i = (tid & 255) >> 3, ch = 16 * (tid & 7), at = mine0 + 32 * nb + i, r = row0 + at;      // a row's 16 channels each
        if (r < late->rows) {
            const float *s0 = buf0 + i * kSumRow + ch, *s1 = s0 + 32 * kSumRow;
            const float total = (sums[at] + sums[M + at]) + (sums[2 * M + at] + sums[3 * M + at]);
            const int64_t head = hkv * late->G + r % late->G, token = r / late->G;
            if (late->part) {
                float *dst = late->part + ((((int64_t)b * late->Hq + head) * late->n + token) * late->nsplit + split) * kPart;
                if (ch == 0) {
                    dst[0] = fmaxf(fmaxf(st[at], st[M + at]), fmaxf(st[2 * M + at], st[3 * M + at]));
                    dst[1] = total;
                }
#pragma unroll
                for (int k = 0; k < 16; k++) dst[4 + ch + k] = s0[k] + s1[k];
            } else {
                const float inv = total == 0.f ? 0.f : 1.f / total;         // (a row that sees no token: zeroes)
                uint32_t o[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float x = (s0[2 * k] + s1[2 * k]) * inv, y = (s0[2 * k + 1] + s1[2 * k + 1]) * inv;
                    o[k] = BF ? pack_bf16(x, y) : pack_f16(x, y);
                }
                u4 *dst = reinterpret_cast<u4 *>(late->out + (int64_t)b * late->o_b + head * late->o_h + token * late->o_t + ch);
                dst[0] = (u4){o[0], o[1], o[2], o[3]};
                dst[1] = (u4){o[4], o[5], o[6], o[7]};
            }
        }
        __syncthreads();
    }
}

// The runs' partials of a row become its result: eight rows a workgroup, four channels a lane.
template <bool BF>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const float *__restrict__ part, uint16_t *__restrict__ out, int64_t rows, int Hq, int n,
                                                          int nsplit, int64_t o_b, int64_t o_h, int64_t o_t) {
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= rows) return;
    const int c = threadIdx.x & 31;
    const float *src = part + r * nsplit * kPart;
    float m = kLowest;
    for (int s = c; s < nsplit; s += 32) m = fmaxf(m, src[(int64_t)s * kPart]);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 32));
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < nsplit; s++) {
        const float *at = src + (int64_t)s * kPart;
        const float f = __builtin_amdgcn_exp2f(at[0] - m);
        const float4 v = *reinterpret_cast<const float4 *>(at + 4 + 4 * c);
        l += f * at[1];
        o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t token = r % n, head = r / n % Hq, b = r / n / Hq;
    uint2 *dst = reinterpret_cast<uint2 *>(out + b * o_b + head * o_h + token * o_t + 4 * c);
    *dst = BF ? make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv))
              : make_uint2(pack_f16(o.x * inv, o.y * inv), pack_f16(o.z * inv, o.w * inv));
}

static bool chunk_wide(const pkv_chunk_args *a) { return a->T_c && (a->k_bits > 4 || a->v_bits > 4); }

// LDS bytes of what is staged, and of a block of either side: a block at any phase, and a last word's reach.
static uint32_t chunk_ring(const pkv_chunk_args *a, int rg, uint32_t &slot_k, uint32_t &slot_v) {
    const bool once = rg == 1 && !chunk_wide(a);
    slot_k = (((uint32_t)k_block_bound(64, a->T_c ? a->k_bits : 2) + 15u) & ~15u) + 32u;
    slot_v = (((uint32_t)v_block_bound(64, a->T_c ? a->v_bits : 2) + 15u) & ~15u) + 32u;
    return once ? 2u * slot_k + 2u * slot_v : 4u * slot_k + 2u * (uint32_t)(rg + 1) * slot_v;
}

// How a call is cut: rows a workgroup (32 NB RG), and runs of tiles, so that the rounds of workgroups the device takes -- three a CU of
// the small kind (wide codes: two, although their LDS leaves one from 6 bits on both sides on: 87 KB, and 105 at 8), one of the large -- times the tiles of a run are fewest; a workgroup's start and end count as two tiles, the merge of
// partials as one.
// Rows of 33 to 64 as one workgroup of two groups against two small ones a KV head against half of a large one: 8 sequences x 10 queries of
// 32 + 8 heads over 8192 tokens 65.7, 72.3, 81.3 us, 1 x 16 over 16384 33.3, 38.8, 39.8; sixteen rows or fewer stand at r16.
// What is staged for two groups, 4 K blocks and 6 V blocks, does not fit with (K, V) widths (3, 8), (4, 7), (4, 8), (5, 7), (5, 8), (7, 5),
// (8, 5) and 6 to 8 on both sides: these take 32 rows a workgroup for any prompt, 1 x 512 queries over 8192 tokens 611 us at (4, 8), 654 at
// (6, 6), where (5, 5) takes 189.
struct ChunkCut {
    int nb, rg, r16, row_tiles, tiles, run, nsplit;
};
static ChunkCut chunk_cut(const pkv_chunk_args *a) {
    ChunkCut c;
    const int64_t rows = (int64_t)a->n * (a->Hq / a->Hkv);
    uint32_t slot_k, slot_v;
    c.rg = rows <= 32 || chunk_ring(a, 2, slot_k, slot_v) > 63u * 1024u ? 1 : 2;     // (copies reach 64 KiB)
    c.nb = c.rg == 1 || rows <= 64 ? 1 : 2;
    c.r16 = rows <= 16 && !chunk_wide(a);                  // 1 x 4 queries of 32 + 8 heads over 131072 tokens 75 us, with 32 rows 82; over 4096 16.5 and 17.3
    const int64_t m = 32 * c.nb * c.rg;
    c.row_tiles = (int)((rows + m - 1) / m);
    c.tiles = a->T_c / kChunkTile + (a->T_w + kChunkTile - 1) / kChunkTile;
    const int64_t groups = (int64_t)a->B * a->Hkv * c.row_tiles, slots = c.rg == 2 ? 256 : chunk_wide(a) ? 512 : 768;
    int64_t best = -1;
    for (int want = 1; want <= c.tiles && want <= 512; want++) {
        const int run = (c.tiles + want - 1) / want, nsplit = (c.tiles + run - 1) / run;
        const int64_t cost = (groups * nsplit + slots - 1) / slots * (run + 2) + (nsplit > 1);
        if (best < 0 || cost < best) { best = cost; c.run = run; c.nsplit = nsplit; }
        if (groups * nsplit >= 4 * slots) break;           // (more rounds of shorter runs gain nothing)
    }
    return c;
}

static int chunk_check(const pkv_chunk_args *a) {
    PKV_REQUIRE(a != nullptr, PKV_ERR_INVALID, "null pointer argument");
    PKV_REQUIRE(a->dtype == PKV_F16 || a->dtype == PKV_BF16, PKV_ERR_UNSUPPORTED, "Unsupported data type");
    PKV_REQUIRE(a->B > 0 && a->Hkv > 0 && a->n > 0 && a->Hq > 0 && a->Hq % a->Hkv == 0, PKV_ERR_INVALID, "Hq must be a multiple of Hkv, all sizes positive");
    PKV_REQUIRE(a->T_c >= 0 && a->T_w >= 0 && (int64_t)a->T_c + a->T_w > 0 && (int64_t)a->T_c + a->T_w < (1ll << 30), PKV_ERR_INVALID, "empty cache");
    PKV_REQUIRE(a->T_c % kChunkTile == 0, PKV_ERR_INVALID, "compressed length must be a multiple of 128 tokens");
    PKV_REQUIRE(!a->causal || a->n <= a->T_c + a->T_w, PKV_ERR_INVALID, "more queries than tokens");
    PKV_REQUIRE((int64_t)a->n * (a->Hq / a->Hkv) < (1ll << 30) && (int64_t)a->B * a->Hkv < (1ll << 24), PKV_ERR_UNSUPPORTED, "batch x queries too large");
    return PKV_OK;
}

}  // namespace pkv

extern "C" {

uint64_t pkv_attn_chunk_workspace(const pkv_chunk_args *a) {
    using namespace pkv;
    if (chunk_check(a)) return 0;
    const int nsplit = chunk_cut(a).nsplit;
    return nsplit > 1 ? (uint64_t)a->B * a->Hq * a->n * nsplit * kPart * sizeof(float) : 0;
}

int pkv_attn_chunk(const pkv_chunk_args *a, void *workspace, uint64_t workspace_bytes, pkv_stream_t s_) {
    using namespace pkv;
    hipStream_t s = (hipStream_t)s_;
    const int bad = chunk_check(a);
    if (bad) return bad;
    PKV_REQUIRE(a->q && a->out, PKV_ERR_INVALID, "null pointer argument");
    uint64_t off = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out);
    for (int i = 0; i < 3; i++) off |= 2u * (uint64_t)(a->q_stride[i] | a->out_stride[i]);
    PKV_REQUIRE((off & 15u) == 0, PKV_ERR_INVALID, "rows of q and out must start on 16-byte boundaries");
    ChunkParams p;
    p.par_stride = a->par_stride ? a->par_stride : a->T_c;
    p.win_stride = a->win_stride ? a->win_stride : a->T_w;
    PKV_REQUIRE(p.par_stride >= a->T_c && p.win_stride >= a->T_w, PKV_ERR_INVALID, "row stride shorter than the row");
    if (a->T_c > 0) {
        PKV_REQUIRE(a->k_stream && a->k_info && a->v_stream && a->v_info && a->k_scale && a->k_zero && a->v_scale && a->v_zero, PKV_ERR_INVALID,
                    "null pointer argument");
        PKV_REQUIRE(a->k_bits >= 2 && a->k_bits <= kMaxBits && a->v_bits >= 2 && a->v_bits <= kMaxBits, PKV_ERR_UNSUPPORTED,
                    "not supported: bits_len outside 2..8");
        PKV_REQUIRE(a->k_bytes > 0 && a->v_bytes > 0 && a->k_bytes < (1ull << 32) - 4 && a->v_bytes < (1ull << 32) - 4, PKV_ERR_INVALID,
                    "stream sizes must be in 1 .. 4 GiB - 5");
        PKV_REQUIRE(((reinterpret_cast<uintptr_t>(a->k_stream) | reinterpret_cast<uintptr_t>(a->v_stream)) & 15u) == 0, PKV_ERR_INVALID,
                    "streams must be 16-byte aligned");
        PKV_REQUIRE((uint64_t)(a->T_c / 64) * (uint64_t)a->B * a->Hkv < (1ull << 31), PKV_ERR_UNSUPPORTED, "batch x tokens too large");
    }
    if (a->T_w > 0)
        PKV_REQUIRE(a->k_win && a->v_win && ((reinterpret_cast<uintptr_t>(a->k_win) | reinterpret_cast<uintptr_t>(a->v_win)) & 15u) == 0, PKV_ERR_INVALID,
                    "window tensors must be present and 16-byte aligned");
    const ChunkCut cut = chunk_cut(a);
    p.row_tiles = cut.row_tiles; p.tiles = cut.tiles; p.run = cut.run; p.nsplit = cut.nsplit;
    const uint64_t need = p.nsplit > 1 ? (uint64_t)a->B * a->Hq * a->n * p.nsplit * kPart * sizeof(float) : 0;
    PKV_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0), PKV_ERR_CAPACITY,
                "the call needs a 16-byte aligned workspace of %llu bytes", (unsigned long long)need);
    p.k_stream = a->k_stream; p.v_stream = a->v_stream; p.k_info = a->k_info; p.v_info = a->v_info;
    p.k_scale = (const uint16_t *)a->k_scale; p.k_zero = (const uint16_t *)a->k_zero;
    p.v_scale = (const uint16_t *)a->v_scale; p.v_zero = (const uint16_t *)a->v_zero;
    p.k_win = (const uint16_t *)a->k_win; p.v_win = (const uint16_t *)a->v_win;
    p.q = (const uint16_t *)a->q; p.out = (uint16_t *)a->out;
    p.part = need ? (float *)workspace : nullptr;
    p.starts = a->starts;
    p.q_b = a->q_stride[0]; p.q_h = a->q_stride[1]; p.q_t = a->q_stride[2];
    p.o_b = a->out_stride[0]; p.o_h = a->out_stride[1]; p.o_t = a->out_stride[2];
    p.k_bytes = a->k_bytes; p.v_bytes = a->v_bytes;
    p.Hq = a->Hq; p.Hkv = a->Hkv; p.BH = a->B * a->Hkv; p.G = a->Hq / a->Hkv; p.n = a->n; p.rows = a->n * p.G;
    p.T_c = a->T_c; p.T_w = a->T_w; p.causal = a->causal != 0;
    p.k_bits = a->T_c ? a->k_bits : 2; p.v_bits = a->T_c ? a->v_bits : 2;
    p.tiles_c = a->T_c / kChunkTile;
    p.sm_log2 = a->sm_scale * kLog2e;
    const uint32_t rg = (uint32_t)cut.rg, m = cut.r16 ? 16u : 32u * (uint32_t)cut.nb * rg, kt = rg * 4u * 32u * kKRow;
    p.ring = chunk_ring(a, cut.rg, p.slot_k, p.slot_v);
    if (p.ring + kt < 4u * rg * 32u * kVRow) p.ring = 4u * rg * 32u * kVRow - kt;      // (the end's sums take less: rg * 2 x 32 x 129 floats)
    const bool wide = chunk_wide(a), bf = a->dtype == PKV_BF16;
    const uint32_t lds = p.ring + kt + rg * (4096u + 2048u) + 8u * m * 4u + m * kQRow;
    const uint64_t groups = ((uint64_t)p.BH * p.nsplit + 7) / 8, wgs = groups * 8 * (uint64_t)p.row_tiles;
    PKV_REQUIRE(wgs < (1ull << 24) / rg, PKV_ERR_UNSUPPORTED, "batch x queries too large");           // (2^32 threads)
#define PKV_CHUNK(bf, nb, rg) {(const void *)attn_chunk_kernel<bf, nb, rg, false>, (const void *)attn_chunk_kernel<bf, nb, rg, true>}
    const void *kernels[2][3][2] = {{PKV_CHUNK(false, 1, 1), PKV_CHUNK(false, 1, 2), PKV_CHUNK(false, 2, 2)},
                                    {PKV_CHUNK(true, 1, 1), PKV_CHUNK(true, 1, 2), PKV_CHUNK(true, 2, 2)}};
#undef PKV_CHUNK
    const void *kernel = kernels[bf][cut.rg - 1 + cut.nb - 1][wide];
    if (cut.r16) kernel = bf ? (const void *)attn_chunk_kernel<true, 1, 1, false, true> : (const void *)attn_chunk_kernel<false, 1, 1, false, true>;
    PKV_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    void *params[] = {&p};
    PKV_HIP_CHECK(hipLaunchKernel(kernel, dim3((unsigned)wgs), dim3(256u * rg), params, lds, s));
    if (need) {
        const int64_t rows = (int64_t)a->B * a->Hq * a->n;
        const dim3 grid((unsigned)((rows + 7) / 8));
        if (bf) chunk_merge_kernel<true><<<grid, 256, 0, s>>>(p.part, p.out, rows, a->Hq, a->n, p.nsplit, p.o_b, p.o_h, p.o_t);
        else chunk_merge_kernel<false><<<grid, 256, 0, s>>>(p.part, p.out, rows, a->Hq, a->n, p.nsplit, p.o_b, p.o_h, p.o_t);
        PKV_HIP_CHECK(hipGetLastError());
    }
    return PKV_OK;
}

}  // extern "C"
