// What the 8-bit operators share: 16-bit values in and out, e4m3 (OCP, largest 448) values and the scales of their blocks.
#pragma once
#include "pkv_common.hpp"

namespace pkv {

constexpr int kBlock8 = 128;                       // values of a row that share a scale
constexpr float kTop8 = 448.f;                     // e4m3's largest
constexpr float kLeast8 = 0x1p-100f;               // what a block's largest value counts as at least: its scale stays a normal number

// Whether [a, b] elements with these strides are memory of their own each: results that are not would be written in any order.
inline bool apart(int64_t a, int64_t a_stride, int64_t b, int64_t b_stride) {
    uint64_t x = a_stride < 0 ? 0 - (uint64_t)a_stride : (uint64_t)a_stride, y = b_stride < 0 ? 0 - (uint64_t)b_stride : (uint64_t)b_stride;
    if (a == 1) return b == 1 || y > 0;
    if (b == 1) return x > 0;
    return x <= y ? x > 0 && x <= (y - 1) / (uint64_t)(a - 1) : y > 0 && y <= (x - 1) / (uint64_t)(b - 1);
}

#ifdef __HIPCC__
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <int DT> __device__ __forceinline__ float wide16(uint32_t w, int i) {
    const uint32_t h = i ? w >> 16 : w & 0xFFFFu;
    return DT == PKV_F16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16);
}
template <int DT> __device__ __forceinline__ uint32_t pair16(float a, float b) {
    if (DT == PKV_F16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, (f16x2){(_Float16)a, (_Float16)b});
    }
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
// The largest of the caller's 16 lanes (a DPP row), in all of them.
__device__ __forceinline__ float row16_max(float v) {
    auto from = [&](auto ctrl) {
        return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    v = fmaxf(v, from(std::integral_constant<int, 0xB1>{}));       // lane ^ 1
    v = fmaxf(v, from(std::integral_constant<int, 0x4E>{}));       // lane ^ 2
    v = fmaxf(v, from(std::integral_constant<int, 0x141>{}));      // 7 - lane of eight
    v = fmaxf(v, from(std::integral_constant<int, 0x140>{}));      // 15 - lane
    return v;
}
// The largest |value| of 16-bit words, two at a time as integers: magnitudes in order, moved up so that infinities and NaN come out negative
// and have no part.  (Three instructions a word; as fp32 numbers, compared and selected one by one, ten, and fp16's conversions twice.)
template <int DT> struct Largest16 {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    static constexpr short kUp = (short)(DT == PKV_F16 ? 0x8000 - 0x7C00 : 0x8000 - 0x7F80);
    s16x2 most = {kUp, kUp};
    __device__ __forceinline__ void take(uint32_t w) {
        most = __builtin_elementwise_max(most, __builtin_bit_cast(s16x2, w & 0x7FFF7FFFu) + (s16x2){kUp, kUp});
    }
    __device__ __forceinline__ float value() const {
        const short m = most[0] > most[1] ? most[0] : most[1];
        return wide16<DT>((uint32_t)(uint16_t)(m - kUp), 0);
    }
};
// |v|, and 0 for infinities and NaN, which have no part in a block's scale.
__device__ __forceinline__ float finite_size(float v) {
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.f;
}
__device__ __forceinline__ float scale_of(float largest) { return fmaxf(largest, kLeast8) / kTop8; }
// Eight values over their block's scale, the fp32 quotients to the nearest e4m3, ties to even.  The product with inv, the hardware's 1 / scale (off by a step,
// a normal number for every scale), may be off by three, which loses the ties: its remainder times inv puts it right, to 2^-43 before its
// rounding, and 16-bit values get the codes of an exact division.  (largest / scale may come out a rounding above 448, which still rounds to
// 448; infinities and NaN become NaN.)  8192 x 4096 by rows 19.4 us, without the remainder 19.3; 4848 x 912 in blocks of 128 rows 6.1 and 5.75.
__device__ __forceinline__ float quotient(float y, float scale, float inv) {
    const float q = y * inv;
    return fmaf(-fmaf(q, scale, -y), inv, q);              // (in these signs -0 stays -0)
}
__device__ __forceinline__ u32x2 codes8(const float y[8], float scale) {
    const float inv = __builtin_amdgcn_rcpf(scale);
    u32x2 r = {0u, 0u};
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = quotient(y[i], scale, inv);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], w, true);
        r[i] = (uint32_t)w;
    }
    return r;
}
#endif

}  // namespace pkv
