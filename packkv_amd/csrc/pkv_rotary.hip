// Head norms and rotary embedding of queries and keys in one pass, positions on one or several axes, and the same for a
// decode step whose keys and values go straight into the cache's 16-bit window.
//
// A row x of 128 channels becomes y = x * rsqrt(mean(x^2) + eps) * w (no norm: y = x), and every pair (y_i, y_{i+64}) is
// turned by theta_i = position[axis(i)] * inv_freq[i]:  (y_i cos - y_{i+64} sin, y_{i+64} cos + y_i sin).  All of it in fp32,
// rounded once when it is stored; the angle is formed and reduced to a fraction of a turn in fp64 pairs, since at position 10^6
// an fp32 angle is off by up to 0.06.  (The chain of library kernels rounds after the norm, the cosines and each product.)
//
// Bound by memory, and by the launch where rows are few: a row is read once and written once.  4 x 2048 tokens of 32 + 8 heads, caches
// cold, 30 us (5.6 TB/s; a large copy 5.2); a decode step's write, 1 to 64 sequences, 5.3 us.  Eight lanes hold a row, each 8 channels of either half (two 16-byte
// loads), so the sum of squares takes three exchanges and both halves of a pair are in one lane; a wavefront holds eight heads
// of a token.  Lane i works out frequency i once for the wavefront, and the eight lanes of a row fetch theirs from LDS.
#include "pkv_block.hpp"
#include "pkv_runtime.hpp"

namespace pkv {

struct RotarySide {
    const uint16_t *in, *w;
    uint16_t *out;
    int64_t in_b, in_h, in_t, out_b, out_h, out_t;
    int heads, groups;                   // groups of eight heads
};
struct RotaryParams {
    RotarySide side[3];                  // q, k, v (v: copied)
    const void *pos;
    const float *inv_freq;
    int64_t pos_a, pos_b, pos_t;
    uint64_t axis[2];                    // two bits a frequency
    uint32_t n, groups, pieces;          // groups of all sides together, and of wavefronts' shares of them
    uint64_t units;                      // tokens x pieces
    int per;                             // groups a wavefront
    float eps;
    int pos64;
};

template <int DT> __device__ __forceinline__ float half_at(uint32_t w, int i) {
    const uint32_t h = i ? w >> 16 : w & 0xFFFFu;
    return DT == PKV_F16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16);
}
template <int DT> __device__ __forceinline__ uint32_t half_pair(float a, float b) {
    if (DT == PKV_F16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, (f16x2){(_Float16)a, (_Float16)b});
    }
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
// Eight channels at p, which lies at a multiple of 16 bytes (WIDE) or at any address of its elements.
template <bool WIDE> __device__ __forceinline__ void load8(const uint16_t *p, uint32_t w[4]) {
    if (WIDE) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
}
template <bool WIDE, bool PAST> __device__ __forceinline__ void store8(uint16_t *p, const uint32_t w[4]) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    if (WIDE) {
        const u32x4 v = {w[0], w[1], w[2], w[3]};
        if (PAST) __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(p));
        else *reinterpret_cast<u32x4 *>(p) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) { p[2 * i] = (uint16_t)w[i]; p[2 * i + 1] = (uint16_t)(w[i] >> 16); }
}

// pos * freq as a fraction of a turn, -1/2 .. 1/2.  The product has up to 53 + 24 bits: its rounding error and that of the
// division by 2 pi go along in a second number, so what is left is right to 24 bits at every position.
__device__ __forceinline__ float turn_fraction(double pos, double freq) {
#pragma clang fp contract(off)
    constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnLow = -0x1.6b01ec5417056p-57;      // 1 / (2 pi), and the rest of it
    const double angle = pos * freq, angle_low = fma(pos, freq, -angle);
    const double hi = angle * kTurn, low = fma(angle, kTurn, -hi) + fma(angle, kTurnLow, angle_low * kTurn);
    const double r = (hi - rint(hi)) + low;
    return (float)(r - rint(r));
}

// One wavefront: `per` groups of eight heads of one token, the next group's rows on their way while one is turned.
// PAST: what is stored does not stay in the caches.
template <int DT, bool WIDE, bool PAST>
__global__ void __launch_bounds__(256, 8) norm_rotary_kernel(const RotaryParams p) {
    __shared__ float2 turn_s[4][64];                         // (cos, sin) by frequency, one table a wavefront
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t unit = (uint64_t)blockIdx.x * 4u + (uint32_t)wave;
    if (unit >= p.units) return;                             // (no barrier below: each wavefront is on its own)
    const uint64_t token = unit / p.pieces;
    const int first = (int)(unit - token * p.pieces) * p.per, last = min(first + p.per, (int)p.groups);
    const int64_t b = (int64_t)(token / p.n), t = (int64_t)(token - (uint64_t)b * p.n);
    const int c = 8 * (lane & 7);
    struct Rows {
        uint16_t *out;
        const uint16_t *w;
        bool mine, turned;
        uint32_t lo[4], hi[4];
    };
    auto load = [&](int g) -> Rows {
        int which = 0;
        while (which < 2 && g >= p.side[which].groups) g -= p.side[which++].groups;
        const RotarySide &s = p.side[which];
        const int h = min(8 * g + (lane >> 3), s.heads - 1); // (idle rows repeat the last head's)
        Rows r;
        r.mine = 8 * g + (lane >> 3) < s.heads;
        r.turned = which < 2;
        r.w = s.w;
        const uint16_t *in = s.in + b * s.in_b + (int64_t)h * s.in_h + t * s.in_t;
        r.out = s.out + b * s.out_b + (int64_t)h * s.out_h + t * s.out_t;
        load8<WIDE>(in + c, r.lo);
        load8<WIDE>(in + 64 + c, r.hi);
        return r;
    };
    Rows next = load(first);
    const int axis = (int)(p.axis[lane >> 5] >> (2 * (lane & 31))) & 3;
    const int64_t at = axis * p.pos_a + b * p.pos_b + t * p.pos_t;
    const double pos = p.pos64 ? (double)reinterpret_cast<const int64_t *>(p.pos)[at] : (double)reinterpret_cast<const int32_t *>(p.pos)[at];
    float sn, cs;
    sincospif(2.f * turn_fraction(pos, (double)p.inv_freq[lane]), &sn, &cs);
    turn_s[wave][lane] = make_float2(cs, sn);
    wave_lds_order();
    float2 turn[8];
#pragma unroll
    for (int i = 0; i < 8; i++) turn[i] = turn_s[wave][c + i];
    for (int g = first; g < last; g++) {
        Rows r = next;
        if (g + 1 < last) next = load(g + 1);
        if (r.turned) {
            float x[8], y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = half_at<DT>(r.lo[i >> 1], i & 1);
                y[i] = half_at<DT>(r.hi[i >> 1], i & 1);
            }
            if (r.w) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) sum += x[i] * x[i] + y[i] * y[i];
                sum += __shfl_xor(sum, 1, 64);
                sum += __shfl_xor(sum, 2, 64);
                sum += __shfl_xor(sum, 4, 64);
                const float scale = 1.f / sqrtf(sum * (1.f / 128.f) + p.eps);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[i] *= scale * half_at<DT>(r.w[c + i], 0);
                    y[i] *= scale * half_at<DT>(r.w[64 + c + i], 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 a = turn[2 * i], d = turn[2 * i + 1];
                const float x0 = x[2 * i], x1 = x[2 * i + 1], y0 = y[2 * i], y1 = y[2 * i + 1];
                r.lo[i] = half_pair<DT>(x0 * a.x - y0 * a.y, x1 * d.x - y1 * d.y);
                r.hi[i] = half_pair<DT>(y0 * a.x + x0 * a.y, y1 * d.x + x1 * d.y);
            }
        }
        if (r.mine) {
            store8<WIDE, PAST>(r.out + c, r.lo);
            store8<WIDE, PAST>(r.out + 64 + c, r.hi);
        }
    }
}

}  // namespace pkv

extern "C" int pkv_norm_rotary(const pkv_rotary_args *a, pkv_stream_t s_) {
    using namespace pkv;
    hipStream_t s = (hipStream_t)s_;
    PKV_REQUIRE(a && a->q && a->k && a->q_out && a->k_out && a->positions && a->inv_freq, PKV_ERR_INVALID, "null pointer argument");
    PKV_REQUIRE((a->v == nullptr) == (a->v_out == nullptr), PKV_ERR_INVALID, "values need an output, and an output values");
    PKV_REQUIRE(a->dtype == PKV_F16 || a->dtype == PKV_BF16, PKV_ERR_UNSUPPORTED, "Unsupported data type");
    PKV_REQUIRE(a->B > 0 && a->Hq > 0 && a->Hkv > 0 && a->n > 0, PKV_ERR_INVALID, "sizes must be positive");
    PKV_REQUIRE(a->pos_bytes == 4 || a->pos_bytes == 8, PKV_ERR_INVALID, "positions are 32- or 64-bit integers");
    PKV_REQUIRE(a->n_axes >= 1 && a->n_axes <= 4, PKV_ERR_UNSUPPORTED, "not supported: %d position axes (1 to 4)", a->n_axes);
    RotaryParams p;
    p.side[0] = RotarySide{(const uint16_t *)a->q, (const uint16_t *)a->q_norm, (uint16_t *)a->q_out, a->q_stride[0], a->q_stride[1], a->q_stride[2],
                           a->q_out_stride[0], a->q_out_stride[1], a->q_out_stride[2], a->Hq, (a->Hq + 7) / 8};
    p.side[1] = RotarySide{(const uint16_t *)a->k, (const uint16_t *)a->k_norm, (uint16_t *)a->k_out, a->k_stride[0], a->k_stride[1], a->k_stride[2],
                           a->k_out_stride[0], a->k_out_stride[1], a->k_out_stride[2], a->Hkv, (a->Hkv + 7) / 8};
    p.side[2] = RotarySide{(const uint16_t *)a->v, nullptr, (uint16_t *)a->v_out, a->v_stride[0], a->v_stride[1], a->v_stride[2],
                           a->v_out_stride[0], a->v_out_stride[1], a->v_out_stride[2], a->Hkv, a->v ? (a->Hkv + 7) / 8 : 0};
    uint64_t off = 0;                    // every address bit below 16 bytes that a row can have
    for (int i = 0; i < (a->v ? 3 : 2); i++) {
        const RotarySide &d = p.side[i];
        off |= reinterpret_cast<uintptr_t>(d.in) | reinterpret_cast<uintptr_t>(d.out) |
               2u * (uint64_t)(d.in_b | d.in_h | d.in_t | d.out_b | d.out_h | d.out_t);
    }
    p.axis[0] = p.axis[1] = 0;
    for (int i = 0; i < 64; i++) {
        PKV_REQUIRE(a->axis[i] < a->n_axes, PKV_ERR_INVALID, "frequency %d belongs to an axis that is not there", i);
        p.axis[i >> 5] |= (uint64_t)a->axis[i] << (2 * (i & 31));
    }
    p.pos = a->positions;
    p.pos64 = a->pos_bytes == 8;
    p.pos_a = a->pos_stride[0]; p.pos_b = a->pos_stride[1]; p.pos_t = a->pos_stride[2];
    p.inv_freq = a->inv_freq;
    p.eps = a->eps;
    p.n = (uint32_t)a->n;
    p.groups = (uint32_t)(p.side[0].groups + p.side[1].groups + p.side[2].groups);
    const uint64_t tokens = (uint64_t)a->B * (uint64_t)a->n;
    // As many groups a wavefront as leave one round of them (32 a CU): the angles are worked out once for all, and rows are on their
    // way meanwhile.  4 x 2048 tokens of 32 + 8 heads, one group -> two, three, five: 39.2 us -> 34.1, 33.3, 31.4 (5.35 TB/s; a
    // large copy 5.2); 2 x 1031 of 16 + 4, which are less than a round: 8.4 -> 8.7, 9.4, 9.4.
    const uint64_t rounds = tokens * p.groups / 8192;
    p.per = (int)(rounds < 1 ? 1 : rounds < p.groups ? rounds : p.groups);
    // Results that no L2 would hold until they are read go past it, where they push out what is still to be read otherwise: 4 x 2048
    // tokens (84 MB of results), caches cold, 37.3 -> 29.8 us, 2 x 1031 (10.5 MB) 7.75 -> 6.52; 64 x 1 (0.8 MB) 5.3 -> 5.4.  (Loads that way
    // too: 32.8, alone 31.4.)
    const bool past = tokens * (uint64_t)(a->Hq + (a->v ? 2 : 1) * a->Hkv) * 256u > (4u << 20);
    p.pieces = (p.groups + (uint32_t)p.per - 1u) / (uint32_t)p.per;
    p.units = tokens * p.pieces;
    const uint64_t wgs = (p.units + 3) / 4;
    PKV_REQUIRE(wgs < (1ull << 24), PKV_ERR_UNSUPPORTED, "batch x tokens x heads too large");         // (2^32 threads)
    const dim3 grid((unsigned)wgs);
    if (off & 15u) {
        if (a->dtype == PKV_F16) norm_rotary_kernel<PKV_F16, false, false><<<grid, 256, 0, s>>>(p);
        else norm_rotary_kernel<PKV_BF16, false, false><<<grid, 256, 0, s>>>(p);
    } else if (past) {
        if (a->dtype == PKV_F16) norm_rotary_kernel<PKV_F16, true, true><<<grid, 256, 0, s>>>(p);
        else norm_rotary_kernel<PKV_BF16, true, true><<<grid, 256, 0, s>>>(p);
    } else {
        if (a->dtype == PKV_F16) norm_rotary_kernel<PKV_F16, true, false><<<grid, 256, 0, s>>>(p);
        else norm_rotary_kernel<PKV_BF16, true, false><<<grid, 256, 0, s>>>(p);
    }
    PKV_HIP_CHECK(hipGetLastError());
    return PKV_OK;
}
