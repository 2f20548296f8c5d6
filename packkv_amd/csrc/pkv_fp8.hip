// Root-mean-square norm of a residual's sum, and the 8-bit form of 16-bit tensors: what the 8-bit products (pkv_fp8_product.hip) read.
//
// The 8-bit form of a matrix y [rows, width] has one fp32 scale for each block of 1 x 128 (activations) or 128 x 128 values
// (weights), the last blocks ragged: s = max(max |y|, 2^-100) / 448, codes e4m3(y / s).  The norm is h = x + residual,
// n = h / sqrt(mean(h^2) + eps) * w, all in fp32 from the sum on; h is rounded once where it is stored, n once to 16 bits or 8.
//
// Bound by memory, and by the launch where rows are few.  A thread holds chunks of eight values (one 16-byte load of each input),
// so sixteen lanes hold a block and its largest value takes four DPP steps.
#include <type_traits>

#include "pkv_fp8.hpp"
#include "pkv_runtime.hpp"

namespace pkv {

struct NormParams {
    const uint16_t *x, *residual, *weight;
    uint16_t *sum, *out;
    uint8_t *codes;
    float *scale;
    int64_t x_row, residual_row, sum_row, out_row, codes_row, scale_row, scale_col;
    uint32_t rows, width;
    float eps;
};

// T threads a row (64: four rows a workgroup), V chunks of eight values a thread.
template <int DT, int T, int V>
__global__ void __launch_bounds__(T < 256 ? 256 : T) norm_kernel(const NormParams p) {
    constexpr int kWaves = T / 64;
    const uint32_t row = T == 64 ? blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
    if (row >= p.rows) return;                             // (T == 64: no barrier below)
    const uint32_t t = threadIdx.x & (T - 1);
    const uint16_t *x = p.x + (int64_t)row * p.x_row, *res = p.residual ? p.residual + (int64_t)row * p.residual_row : nullptr;
    float h[V][8];
    float sum = 0.f;
    u32x4_t xs[V], rs[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t c = 8u * (t + (uint32_t)(i * T));
        xs[i] = rs[i] = (u32x4_t){0u, 0u, 0u, 0u};
        if (c < p.width) {
            xs[i] = *reinterpret_cast<const u32x4_t *>(x + c);
            if (res) rs[i] = *reinterpret_cast<const u32x4_t *>(res + c);
        }
    }
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            h[i][j] = wide16<DT>(xs[i][j >> 1], j & 1);
            if (res) h[i][j] += wide16<DT>(rs[i][j >> 1], j & 1);
            sum += h[i][j] * h[i][j];
        }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
    if (kWaves > 1) {
        __shared__ float part[kWaves > 1 ? kWaves : 1];
        if ((t & 63u) == 0) part[t >> 6] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) sum += part[w];
    }
    const float size = 1.f / sqrtf(sum / (float)p.width + p.eps);
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t c = 8u * (t + (uint32_t)(i * T));
        float y[8], most = 0.f;
        const bool mine = c < p.width;                     // (a block's lanes behind the width take part with zeroes)
        if (mine) {
            if (p.sum) {
                u32x4_t v;
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = pair16<DT>(h[i][2 * j], h[i][2 * j + 1]);
                *reinterpret_cast<u32x4_t *>(p.sum + (int64_t)row * p.sum_row + c) = v;
            }
            const u32x4_t w = *reinterpret_cast<const u32x4_t *>(p.weight + c);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                y[j] = h[i][j] * size * wide16<DT>(w[j >> 1], j & 1);
                most = fmaxf(most, finite_size(y[j]));
            }
        }
        if (p.codes) {
            const float s = scale_of(row16_max(most));
            if (mine) {
                *reinterpret_cast<u32x2 *>(p.codes + (int64_t)row * p.codes_row + c) = codes8(y, s);
                if ((t & 15u) == 0) p.scale[(int64_t)row * p.scale_row + (int64_t)(c / kBlock8) * p.scale_col] = s;
            }
        } else if (mine) {
            u32x4_t v;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = pair16<DT>(y[2 * j], y[2 * j + 1]);
            *reinterpret_cast<u32x4_t *>(p.out + (int64_t)row * p.out_row + c) = v;
        }
    }
}

struct QuantizeParams {
    const uint16_t *x;
    uint8_t *codes;
    float *scale;
    int64_t x_batch, x_row, x_col, codes_row, scale_row, scale_col;      // x_col: from a block of 128 to the next
    uint32_t per_batch, rows, width, cols;                 // cols: blocks of a row
};

// Blocks of 1 x 128, sixteen lanes each: a workgroup has 16 rows and eight blocks of each, a thread one row's, all eight loads on their way at
// once.  (Sixteen rows, so that their scales are whole lines where those of a column lie together: 8192 x 4096 18.6 us, 5.4 TB/s; without the
// remainders of codes8 18.4, and then with rows of 128 blocks 19.6.)
template <int DT>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantizeParams p) {
    constexpr int V = 8;
    const uint32_t lane = threadIdx.x & 15u, across = (p.cols + V - 1u) / V, down = blockIdx.x / across;
    const uint32_t row = down * 16u + (threadIdx.x >> 4), col = (blockIdx.x - down * across) * V;
    if (row >= p.rows) return;                             // (sixteen lanes together, as the exchange below)
    const uint32_t batch = row / p.per_batch;
    const uint16_t *x = p.x + batch * p.x_batch + (int64_t)(row - batch * p.per_batch) * p.x_row;
    u32x4_t v[V];
#pragma unroll
    for (int i = 0; i < V; i++) {                          // (behind the width the block's first chunk again, of blocks behind it the row's)
        const uint32_t b = col + i < p.cols ? col + i : 0u;
        v[i] = *reinterpret_cast<const u32x4_t *>(x + (int64_t)b * p.x_col + (b * kBlock8 + 8u * lane < p.width ? 8u * lane : 0u));
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        Largest16<DT> most;
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; j++) most.take(v[i][j]);
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = wide16<DT>(v[i][j >> 1], j & 1);
        const float s = scale_of(row16_max(most.value()));
        if ((col + i) * kBlock8 + 8u * lane < p.width) {
            *reinterpret_cast<u32x2 *>(p.codes + (int64_t)row * p.codes_row + (col + i) * kBlock8 + 8u * lane) = codes8(y, s);
            if (lane == 0) p.scale[(int64_t)row * p.scale_row + (int64_t)(col + i) * p.scale_col] = s;
        }
    }
}

// Blocks of 128 x 128, one a workgroup: a thread holds eight rows' chunks, so x is read once.  24576 x 4096 54 us (5.6 TB/s; 50 without
// the remainders of codes8), 4848 x 912 6.1 us: one round of 304 workgroups; with 512 threads of four chunks the same.
template <int DT>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const QuantizeParams p) {
    __shared__ float part[4];
    const uint32_t down = blockIdx.x / p.cols, col = blockIdx.x - down * p.cols;
    const uint32_t c = col * kBlock8 + 8u * (threadIdx.x & 15u), first = down * kBlock8 + (threadIdx.x >> 4);
    u32x4_t x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {                          // (behind the last row that row again, behind the width the block's first chunk)
        const uint32_t row = first + (uint32_t)i * 16u;
        x[i] = *reinterpret_cast<const u32x4_t *>(p.x + (int64_t)(row < p.rows ? row : p.rows - 1u) * p.x_row + (c < p.width ? c : col * kBlock8));
    }
    Largest16<DT> sizes;
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) sizes.take(x[i][j]);
    float most = sizes.value();
#pragma unroll
    for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d, 64));
    if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
    const float s = scale_of(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
    if (threadIdx.x == 0) p.scale[(int64_t)down * p.scale_row + (int64_t)col * p.scale_col] = s;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t row = first + (uint32_t)i * 16u;
        if (row < p.rows && c < p.width) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = wide16<DT>(x[i][j >> 1], j & 1);
            *reinterpret_cast<u32x2 *>(p.codes + (int64_t)row * p.codes_row + c) = codes8(y, s);
        }
    }
}

// A wavefront a row (no barrier) where there are rows enough to fill the card with and a thread has 32 values at most, 256 or 1024 threads
// a row otherwise.  8192 x 4096 with a residual, 8 bits out: 64 threads of 64 values 100 us (their sums leave two wavefronts a SIMD), 256 of 16 44.2 (5.3 TB/s; a
// large copy 5.1); 16384 x 2048, 64 of 32 44.5; 2048 x 16384, 1024 of 16 44.5.
template <int DT> void launch_norm(const NormParams &p, hipStream_t s) {
    const uint32_t w = p.width;
    const dim3 fours((p.rows + 3) / 4), ones(p.rows);
    if (p.rows >= 1024 && w <= 2048) {                     // a wavefront a row
        if (w <= 512) norm_kernel<DT, 64, 1><<<fours, 256, 0, s>>>(p);
        else if (w <= 1024) norm_kernel<DT, 64, 2><<<fours, 256, 0, s>>>(p);
        else norm_kernel<DT, 64, 4><<<fours, 256, 0, s>>>(p);
    } else if (w <= 2048) norm_kernel<DT, 256, 1><<<ones, 256, 0, s>>>(p);
    else if (w <= 4096) norm_kernel<DT, 256, 2><<<ones, 256, 0, s>>>(p);
    else if (w <= 8192) norm_kernel<DT, 256, 4><<<ones, 256, 0, s>>>(p);
    else if (w <= 16384) norm_kernel<DT, 1024, 2><<<ones, 1024, 0, s>>>(p);
    else if (w <= 32768) norm_kernel<DT, 1024, 4><<<ones, 1024, 0, s>>>(p);
    else norm_kernel<DT, 1024, 8><<<ones, 1024, 0, s>>>(p);
}

}  // namespace pkv

extern "C" int pkv_add_rms_norm(const pkv_norm_args *a, pkv_stream_t s_) {
    using namespace pkv;
    hipStream_t s = (hipStream_t)s_;
    PKV_REQUIRE(a && a->x && a->weight, PKV_ERR_INVALID, "null pointer argument");
    PKV_REQUIRE((a->residual == nullptr) == (a->sum == nullptr), PKV_ERR_INVALID, "a residual needs an output for the sum, and the sum a residual");
    PKV_REQUIRE((a->out == nullptr) != (a->codes == nullptr) && (a->codes == nullptr) == (a->scale == nullptr), PKV_ERR_INVALID,
                "the result goes to out, or to codes and scale");
    PKV_REQUIRE(a->dtype == PKV_F16 || a->dtype == PKV_BF16, PKV_ERR_UNSUPPORTED, "Unsupported data type");
    PKV_REQUIRE(a->rows > 0 && a->width > 0, PKV_ERR_INVALID, "sizes must be positive");
    PKV_REQUIRE(a->width % 16 == 0 && a->width <= 65536, PKV_ERR_UNSUPPORTED, "not supported: width %d (multiples of 16 up to 65536)", a->width);
    PKV_REQUIRE(a->rows < (1 << 22), PKV_ERR_UNSUPPORTED, "not supported: %d rows (fewer than 2^22)", a->rows);        // (2^32 threads)
    const uintptr_t off = (uintptr_t)a->x | (uintptr_t)a->residual | (uintptr_t)a->weight | (uintptr_t)a->sum | (uintptr_t)a->out | (uintptr_t)a->codes |
                          (uintptr_t)(2 * (a->x_stride | a->residual_stride | a->sum_stride | a->out_stride)) | (uintptr_t)a->codes_stride;
    PKV_REQUIRE(off % 16 == 0 && (uintptr_t)a->scale % 4 == 0, PKV_ERR_INVALID, "rows must start on 16-byte boundaries");
    const int cols = (a->width + kBlock8 - 1) / kBlock8;
    PKV_REQUIRE((!a->sum || apart(a->rows, a->sum_stride, a->width, 1)) && apart(a->rows, a->out ? a->out_stride : a->codes_stride, a->width, 1) &&
                (!a->scale || apart(a->rows, a->scale_stride[0], cols, a->scale_stride[1])), PKV_ERR_INVALID, "results must not overlap");
    NormParams p;
    p.x = (const uint16_t *)a->x; p.residual = (const uint16_t *)a->residual; p.weight = (const uint16_t *)a->weight;
    p.sum = (uint16_t *)a->sum; p.out = (uint16_t *)a->out; p.codes = a->codes; p.scale = a->scale;
    p.x_row = a->x_stride; p.residual_row = a->residual_stride; p.sum_row = a->sum_stride; p.out_row = a->out_stride; p.codes_row = a->codes_stride;
    p.scale_row = a->scale_stride[0]; p.scale_col = a->scale_stride[1];
    p.rows = (uint32_t)a->rows; p.width = (uint32_t)a->width;
    p.eps = a->eps;
    if (a->dtype == PKV_F16) launch_norm<PKV_F16>(p, s);
    else launch_norm<PKV_BF16>(p, s);
    PKV_HIP_CHECK(hipGetLastError());
    return PKV_OK;
}

extern "C" int pkv_fp8_quantize(const pkv_fp8_quantize_args *a, pkv_stream_t s_) {
    using namespace pkv;
    hipStream_t s = (hipStream_t)s_;
    PKV_REQUIRE(a && a->x && a->codes && a->scale, PKV_ERR_INVALID, "null pointer argument");
    PKV_REQUIRE(a->dtype == PKV_F16 || a->dtype == PKV_BF16, PKV_ERR_UNSUPPORTED, "Unsupported data type");
    PKV_REQUIRE(a->rows > 0 && a->width > 0 && a->per_batch > 0, PKV_ERR_INVALID, "sizes must be positive");
    PKV_REQUIRE(a->width % 16 == 0, PKV_ERR_UNSUPPORTED, "not supported: width %d (multiples of 16)", a->width);
    PKV_REQUIRE(a->block == 1 || a->block == kBlock8, PKV_ERR_UNSUPPORTED, "not supported: blocks of %d rows (1 or 128)", a->block);
    PKV_REQUIRE(a->block == 1 || (a->per_batch >= a->rows && a->x_stride[2] == kBlock8), PKV_ERR_UNSUPPORTED, "not supported: heads in blocks of 128 rows");
    const uintptr_t off = (uintptr_t)a->x | (uintptr_t)a->codes | (uintptr_t)(2 * (a->x_stride[0] | a->x_stride[1] | a->x_stride[2])) | (uintptr_t)a->codes_stride;
    PKV_REQUIRE(off % 16 == 0 && (uintptr_t)a->scale % 4 == 0, PKV_ERR_INVALID, "rows must start on 16-byte boundaries");
    QuantizeParams p;
    p.x = (const uint16_t *)a->x; p.codes = a->codes; p.scale = a->scale;
    p.x_batch = a->x_stride[0]; p.x_row = a->x_stride[1]; p.x_col = a->x_stride[2]; p.codes_row = a->codes_stride;
    p.scale_row = a->scale_stride[0]; p.scale_col = a->scale_stride[1];
    p.per_batch = (uint32_t)a->per_batch; p.rows = (uint32_t)a->rows; p.width = (uint32_t)a->width;
    p.cols = (p.width + kBlock8 - 1) / kBlock8;
    const uint64_t wgs = a->block == 1 ? ((uint64_t)p.rows + 15) / 16 * ((p.cols + 7) / 8) : ((uint64_t)p.rows + kBlock8 - 1) / kBlock8 * p.cols;
    PKV_REQUIRE(wgs < (1ull << 24), PKV_ERR_UNSUPPORTED, "rows x width too large");                // (2^32 threads)
    PKV_REQUIRE(apart(a->rows, a->codes_stride, a->width, 1) && apart((a->rows - 1) / a->block + 1, a->scale_stride[0], p.cols, a->scale_stride[1]),
                PKV_ERR_INVALID, "results must not overlap");
    const dim3 grid((unsigned)wgs);
    if (a->block == 1) {
        if (a->dtype == PKV_F16) quantize_rows_kernel<PKV_F16><<<grid, 256, 0, s>>>(p);
        else quantize_rows_kernel<PKV_BF16><<<grid, 256, 0, s>>>(p);
    } else {
        if (a->dtype == PKV_F16) quantize_blocks_kernel<PKV_F16><<<grid, 256, 0, s>>>(p);
        else quantize_blocks_kernel<PKV_BF16><<<grid, 256, 0, s>>>(p);
    }
    PKV_HIP_CHECK(hipGetLastError());
    return PKV_OK;
}
