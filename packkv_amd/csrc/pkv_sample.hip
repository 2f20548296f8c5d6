// A token for each row of logits from a given uniform number: temperature, top-k, top-p, min-p, and the draw.
//
// Order of a row: logit descending, equal logits by index.  Weight of a token: e = 2^a, a = (logit - max) log2(e) / T.  Each filter
// keeps a prefix of the order -- the first k; the tokens with less than p of the k's mass before them; those with e >= min_p -- and
// the draw takes the first token whose inclusive mass exceeds u times the mass kept.  So nothing is sorted as a whole: a histogram
// of the row over 2048 bins of a (1/48 each, counts and masses) says in which bins a filter can end and in which the draw can fall;
// only those bins' tokens are gathered, ordered and looked at one by one.
//
// Exact whatever the order of the additions: weights are formed in fp64 and held as integers of 2^-43, their sums are whole numbers
// (below 2^63 for 2^20 tokens), so a row gives the same token from any number of workgroups.  Two tokens of a row of 150000 are told
// apart at 10^-13 of its mass, against 2^-24 of the uniform numbers.
#include "pkv_block.hpp"
#include "pkv_runtime.hpp"

namespace pkv {

constexpr int kSampThreads = 1024, kBins = 2048, kCand = 2048, kFracBits = 43;
constexpr double kBinsPerUnit = 48.0;
constexpr int kF32 = 2;                                    // (beside PKV_F16 and PKV_BF16)

struct SampleParams {
    const void *logits;
    const float *u, *temperature, *top_p, *min_p;          // NULL (but u): the numbers below for every row
    const int32_t *top_k;
    int64_t *token;
    float *logprob;
    int64_t row_stride;
    int rows, vocab, top_k_all;
    float temperature_all, top_p_all, min_p_all;
};

// A row's filters.
struct RowRule {
    double per_unit, top_p, min_a, u;                      // a = (x - max) * per_unit; tokens need a >= min_a
    uint32_t top_k;                                        // 0: off
    bool by_p, by_min;
};
__device__ __forceinline__ RowRule row_rule(const SampleParams &p, int row) {
    RowRule r;
    float t = p.temperature ? p.temperature[row] : p.temperature_all;
    const float top = p.top_p ? p.top_p[row] : p.top_p_all, least = p.min_p ? p.min_p[row] : p.min_p_all;
    const int k = p.top_k ? p.top_k[row] : p.top_k_all;
    r.top_k = k > 0 ? (uint32_t)k : 0u;
    if (!(t > 0.f)) { t = 1.f; r.top_k = 1; }              // temperature 0: the first of the order
    r.per_unit = 1.4426950408889634074 / (double)t;
    r.by_p = top < 1.f;
    r.top_p = fmax((double)top, 0.0);
    r.by_min = least > 0.f;
    r.min_a = r.by_min ? fmin(log2((double)least), 0.0) : 0.0;
    r.u = fmin(fmax((double)p.u[row], 0.0), 1.0 - 0x1p-30);
    return r;
}
__device__ __forceinline__ double exponent_of(float x, float top, const RowRule &r) {
    return x == top ? 0.0 : fmax(((double)x - (double)top) * r.per_unit, -1.0e9);
}
__device__ __forceinline__ int bin_of(double a) { return (int)fmin(a * -kBinsPerUnit, (double)(kBins - 1)); }
// 2^a as a whole number of 2^-43, a <= 0: the series of 2^f around 0, |f| <= 1/2, to f^11 / 11! (the rest is below 2^-47).
__device__ __forceinline__ uint64_t weight_of(double a) {
    a = fmax(a, -100.0);
    const double k = rint(a), f = a - k;
    double s = 4.4455382718708114976e-10;
    s = fma(s, f, 7.0549116208011233299e-09);
    s = fma(s, f, 1.0178086009239699728e-07);
    s = fma(s, f, 1.3215486790144309488e-06);
    s = fma(s, f, 1.5252733804059840280e-05);
    s = fma(s, f, 1.5403530393381609954e-04);
    s = fma(s, f, 1.3333558146428443423e-03);
    s = fma(s, f, 9.6181291076284771619e-03);
    s = fma(s, f, 5.5504108664821579953e-02);
    s = fma(s, f, 2.4022650695910071233e-01);
    s = fma(s, f, 6.9314718055994530942e-01);
    s = fma(s, f, 1.0);
    const double fixed = ldexp(s, (int)k + kFracBits) + 0x1p52;              // (the low bits of the sum are the rounded number)
    return (uint64_t)__double_as_longlong(fixed) & ((1ull << 52) - 1ull);
}
// Ascending order of (logit descending, index ascending); x is finite or +inf and not -0.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t idx) {
    const uint32_t b = __float_as_uint(x);
    return ((uint64_t)~(b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u)) << 32) | idx;
}
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t b = ~(uint32_t)(key >> 32);
    return __uint_as_float(b ^ ((b >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

// f(index, logit) for the row's tokens that can be chosen in 16-byte pieces from .. to - 1 (piece 0 holds the row's first logit): the
// pieces are aligned, so the first and the last may hold others' bytes as well, which are not looked at.  -inf and NaN are left out.
template <int DT> __device__ __forceinline__ int row_pieces(const SampleParams &p, int row, const uint4 *&base, int &phase) {
    constexpr int ES = DT == kF32 ? 4 : 2;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.logits) + (uintptr_t)((int64_t)row * p.row_stride) * ES;
    base = reinterpret_cast<const uint4 *>(at & ~(uintptr_t)15);
    phase = (int)(at & 15) / ES;
    return (phase + p.vocab + 16 / ES - 1) / (16 / ES);
}
template <int DT, class F>
__device__ __forceinline__ void for_tokens(const SampleParams &p, const uint4 *base, int phase, int from, int to, F f) {
    constexpr int N = DT == kF32 ? 4 : 8;
    for (int c = from + (int)threadIdx.x; c < to; c += kSampThreads) {
        const uint4 v = base[c];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < N; e++) {
            float x;
            if (DT == kF32) x = __uint_as_float(w[e]);
            else {
                const uint32_t half = (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
                x = DT == PKV_F16 ? __half2float(__ushort_as_half((unsigned short)half)) : __uint_as_float(half << 16);
            }
            const int idx = c * N + e - phase;
            if ((uint32_t)idx < (uint32_t)p.vocab && x > -INFINITY) f((uint32_t)idx, x + 0.f);       // (+ 0: -0 equals 0)
        }
    }
}

// What the launches of a split call hand on, in the workspace: one of these a row.
constexpr int kMaxSlices = 64;
struct RowState {
    uint64_t mass[kBins], cand[kCand];
    uint32_t count[kBins], need[kBins / 32];
    float slice_top[kMaxSlices];
    uint32_t n_need, n_cand, arrived[2];
};
template <class T> __device__ __forceinline__ T far_load(const T *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class T> __device__ __forceinline__ void far_store(T *p, T x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct Prefix { uint64_t mass; uint32_t count; };

// What a row's resolution keeps in LDS.
struct SampleLds {
    uint64_t mass[kBins];                                  // of the bin; after scan(): up to and with the bin
    uint32_t count[kBins];
    uint64_t cand[kCand];
    uint64_t wave_mass[16];
    uint32_t wave_count[16];
    uint32_t need[kBins / 32];
    float top;
    uint32_t n_cand;
    uint64_t best, sums[3];
    int at[4];
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
    return ((uint64_t)(uint32_t)__shfl_up((int)(uint32_t)(v >> 32), d, 64) << 32) | (uint32_t)__shfl_up((int)(uint32_t)v, d, 64);
}
// Inclusive sums over the workgroup's 1024 threads.
__device__ __forceinline__ Prefix block_scan(SampleLds &s, Prefix v) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t m = shfl_up64(v.mass, d);
        const uint32_t c = (uint32_t)__shfl_up((int)v.count, d, 64);
        if (lane >= d) { v.mass += m; v.count += c; }
    }
    __syncthreads();
    if (lane == 63) { s.wave_mass[wave] = v.mass; s.wave_count[wave] = v.count; }
    __syncthreads();
    for (int w = 0; w < wave; w++) { v.mass += s.wave_mass[w]; v.count += s.wave_count[w]; }
    return v;
}
// The histogram becomes inclusive sums.
__device__ __forceinline__ void scan_bins(SampleLds &s) {
    const int b = 2 * threadIdx.x;
    const uint64_t m0 = s.mass[b], m1 = s.mass[b + 1];
    const uint32_t c0 = s.count[b], c1 = s.count[b + 1];
    const Prefix v = block_scan(s, Prefix{m0 + m1, c0 + c1});
    s.mass[b] = v.mass - m1; s.mass[b + 1] = v.mass;
    s.count[b] = v.count - c1; s.count[b + 1] = v.count;
    __syncthreads();
}
// The first bin whose inclusive sum satisfies the condition (kBins: none).  Every thread of the workgroup calls it.
template <class F> __device__ __forceinline__ int first_bin(SampleLds &s, F holds) {
    __syncthreads();
    if (threadIdx.x == 0) s.at[0] = kBins;
    __syncthreads();
    const int b = 2 * threadIdx.x;
    const bool h0 = holds(b), h1 = holds(b + 1);
    if (h0 && (b == 0 || !holds(b - 1))) s.at[0] = b;
    else if (h1 && !h0) s.at[0] = b + 1;
    __syncthreads();
    return s.at[0];
}
__device__ __forceinline__ uint64_t mass_before(const SampleLds &s, int bin) { return bin ? s.mass[bin - 1] : 0ull; }
__device__ __forceinline__ uint32_t count_before(const SampleLds &s, int bin) { return bin ? s.count[bin - 1] : 0u; }

// Where the filters can end, from the scanned histogram.
struct Cuts {
    uint32_t n;                                            // tokens that can be chosen
    int k_bin;                                             // top-k: ends inside this bin (k_inside) or before it; kBins: nowhere
    bool k_inside;
    int low, high;                                         // the bins that the last kept token can be in (kBins: every token is kept)
};
__device__ __forceinline__ Cuts find_cuts(SampleLds &s, const RowRule &r) {
    Cuts c;
    c.n = s.count[kBins - 1];
    c.k_bin = kBins;
    c.k_inside = false;
    uint64_t k_low = s.mass[kBins - 1], k_high = k_low;    // mass of the k tokens, between these
    if (r.top_k && r.top_k < c.n) {
        const int b = first_bin(s, [&](int i) { return s.count[i] >= r.top_k; });
        c.k_inside = s.count[b] != r.top_k;
        c.k_bin = c.k_inside ? b : b + 1;
        k_low = c.k_inside ? mass_before(s, b) : s.mass[b];
        k_high = s.mass[b];
    }
    c.low = c.high = c.k_bin;
    if (r.by_p) {
        const double low = r.top_p * (double)k_low, high = r.top_p * (double)k_high;
        c.low = min(c.low, first_bin(s, [&](int i) { return s.count[i] && (double)s.mass[i] >= low; }));
        c.high = min(c.high, first_bin(s, [&](int i) { return s.count[i] && (double)s.mass[i] >= high; }));
    }
    if (r.by_min) {
        const int b = bin_of(r.min_a);
        c.low = min(c.low, b);
        c.high = min(c.high, b);
    }
    return c;
}
__device__ __forceinline__ void need_bins(SampleLds &s, int from, int to) {              // one thread
    for (int b = from; b <= min(to, kBins - 1); b++) s.need[b >> 5] |= 1u << (b & 31);
}
// Marks the bins whose tokens the answer depends on one by one.
__device__ __forceinline__ void mark_bins(SampleLds &s, const RowRule &r, const Cuts &c) {
    const uint64_t low = c.low < kBins ? max(mass_before(s, c.low), 1ull << kFracBits) : s.mass[kBins - 1];
    const uint64_t high = c.high >= kBins ? s.mass[kBins - 1] : c.high == c.k_bin && !c.k_inside ? mass_before(s, c.high) : s.mass[c.high];
    const double from = r.u * (double)low, to = r.u * (double)max(low, high);
    const int d0 = first_bin(s, [&](int i) { return (double)s.mass[i] > from; }), d1 = first_bin(s, [&](int i) { return (double)s.mass[i] > to; });
    if (threadIdx.x < kBins / 32) s.need[threadIdx.x] = 0u;
    __syncthreads();
    if (threadIdx.x == 0) {
        if (c.k_inside) need_bins(s, c.k_bin, c.k_bin);
        if (r.by_p || r.by_min) need_bins(s, c.low, c.high == c.k_bin && !c.k_inside ? c.high - 1 : c.high);
        need_bins(s, d0, d1);
    }
    __syncthreads();
}
__device__ __forceinline__ bool needed(const SampleLds &s, int bin) { return (s.need[bin >> 5] >> (bin & 31)) & 1u; }

__device__ __forceinline__ void sort_candidates(SampleLds &s, uint32_t n) {
    uint32_t size = 64;
    while (size < n) size <<= 1;
    for (uint32_t i = n + threadIdx.x; i < size; i += kSampThreads) s.cand[i] = ~0ull;
    for (uint32_t k = 2; k <= size; k <<= 1)
        for (uint32_t j = k >> 1; j; j >>= 1) {
            __syncthreads();
            for (uint32_t t = threadIdx.x; t < size / 2; t += kSampThreads) {
                const uint32_t i = ((t & ~(j - 1)) << 1) | (t & (j - 1));
                const uint64_t a = s.cand[i], b = s.cand[i + j];
                if ((a > b) == ((i & k) == 0)) { s.cand[i] = b; s.cand[i + j] = a; }
            }
        }
    __syncthreads();
}

__device__ __forceinline__ void answer(const SampleParams &p, int row, uint64_t key, float top, const RowRule &r, uint64_t kept) {
    p.token[row] = (int64_t)(uint32_t)key;
    if (p.logprob) p.logprob[row] = (float)((exponent_of(key_logit(key), top, r) - (log2((double)kept) - kFracBits)) * 0.69314718055994530942);
}

// The answer from at most kCand gathered tokens.  A candidate's rank and the mass in front of it are its bin's plus those of the
// candidates of its bin in front of it.
__device__ __forceinline__ void resolve_few(SampleLds &s, const SampleParams &p, int row, const RowRule &r, const Cuts &c, uint32_t n) {
    sort_candidates(s, n);
    uint64_t key[2] = {~0ull, ~0ull}, w[2] = {0, 0}, before[2] = {0, 0};
    uint32_t rank[2] = {0, 0};
    double a[2] = {0, 0};
    int bin[2] = {0, 0};
    const uint32_t i0 = 2 * threadIdx.x;
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (i0 + e < n) {
            key[e] = s.cand[i0 + e];
            a[e] = exponent_of(key_logit(key[e]), s.top, r);
            w[e] = weight_of(a[e]);
            bin[e] = bin_of(a[e]);
        }
    const Prefix v = block_scan(s, Prefix{w[0] + w[1], 0u});
    const uint64_t sum[2] = {v.mass - w[1] - w[0], v.mass - w[1]};         // of the candidates in front
    // where the bin's first candidate stands: a chain of candidates of one bin covers the bin, so its start is found by its count
    __syncthreads();
    uint64_t *sums = s.cand;                                              // (the keys are in registers)
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (i0 + e < n) sums[i0 + e] = sum[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (i0 + e < n) {
            uint32_t lo = 0;                                               // candidates of needed bins in front of this bin
            for (int q = 0; q < (bin[e] >> 5); q++) {
                uint32_t bits = s.need[q];
                while (bits) { const int b = 32 * q + __ffs((int)bits) - 1; lo += s.count[b] - count_before(s, b); bits &= bits - 1; }
            }
            uint32_t bits = s.need[bin[e] >> 5] & ((1u << (bin[e] & 31)) - 1u);
            while (bits) { const int b = 32 * (bin[e] >> 5) + __ffs((int)bits) - 1; lo += s.count[b] - count_before(s, b); bits &= bits - 1; }
            rank[e] = count_before(s, bin[e]) + (i0 + e - lo);
            before[e] = mass_before(s, bin[e]) + (sum[e] - sums[lo]);
        }
    // mass of the k tokens
    if (threadIdx.x == 0) {
        s.sums[0] = c.k_bin >= kBins ? s.mass[kBins - 1] : mass_before(s, c.k_bin);
        s.sums[1] = c.low < kBins ? mass_before(s, c.low) : s.mass[kBins - 1];
        s.best = ~0ull;
        s.sums[2] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (i0 + e < n && c.k_inside && rank[e] + 1 == r.top_k) s.sums[0] = before[e] + w[e];
    __syncthreads();
    const double limit = r.by_p ? r.top_p * (double)s.sums[0] : 0.0;
    bool kept[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        kept[e] = i0 + e < n && (c.k_bin >= kBins || rank[e] < r.top_k) && (!r.by_p || rank[e] == 0 || (double)before[e] < limit) &&
                  (!r.by_min || a[e] >= r.min_a);
        if (kept[e]) atomicMax((unsigned long long *)&s.sums[1], (unsigned long long)(before[e] + w[e]));
    }
    __syncthreads();
    const uint64_t total = s.sums[1];
    const double target = r.u * (double)total;
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (kept[e] && (double)(before[e] + w[e]) > target) atomicMin((unsigned long long *)&s.best, (unsigned long long)key[e]);
    __syncthreads();
    if (threadIdx.x == 0) answer(p, row, s.best, s.top, r, total);
}

// ---- the answer when the bins in question hold more tokens than that (long runs of equal logits): by digits of the order ----
// The token at which a sum of the order first reaches what is asked for, among those of one bin: five passes over the row, each a
// histogram of the next digit (11 + 11 + 10 bits of the logit, 10 + 10 of the index) of the tokens that share the digits so far.
template <int DT, class F>
__device__ __forceinline__ uint64_t descend(SampleLds &s, uint64_t *hist_mass, uint32_t *hist_count, const SampleParams &p, int row, const RowRule &r,
                                            int bin, Prefix &before, F reached) {
    const uint4 *base;
    int phase;
    const int pieces = row_pieces<DT>(p, row, base, phase);
    uint64_t prefix = 0;
    before = Prefix{mass_before(s, bin), count_before(s, bin)};
    constexpr int kShift[5] = {53, 42, 32, 10, 0}, kWidth[5] = {11, 11, 10, 10, 10};
    for (int level = 0; level < 5; level++) {
        const int shift = kShift[level], above = shift + kWidth[level];
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kSampThreads) { hist_mass[i] = 0; hist_count[i] = 0; }
        __syncthreads();
        for_tokens<DT>(p, base, phase, 0, pieces, [&](uint32_t idx, float x) {
            const double a = exponent_of(x, s.top, r);
            if (bin_of(a) != bin) return;
            uint64_t key = order_key(x, idx);
            if (above < 64 && (key >> above) != (prefix >> above)) return;
            const int digit = (int)((key >> shift) & ((1u << kWidth[level]) - 1u));
            atomicAdd((unsigned long long *)&hist_mass[digit], (unsigned long long)weight_of(a));
            atomicAdd(&hist_count[digit], 1u);
        });
        __syncthreads();
        if (threadIdx.x == 0) { s.at[1] = 0; s.at[2] = 0; }
        __syncthreads();
        const int d = 2 * threadIdx.x;
        const uint64_t m0 = hist_mass[d], m1 = hist_mass[d + 1];
        const uint32_t c0 = hist_count[d], c1 = hist_count[d + 1];
        const Prefix v = block_scan(s, Prefix{m0 + m1, c0 + c1});
        const Prefix in[2] = {{before.mass + v.mass - m1, before.count + v.count - c1}, {before.mass + v.mass, before.count + v.count}};
        const Prefix out[2] = {{in[0].mass - m0, in[0].count - c0}, {in[1].mass - m1, in[1].count - c1}};
        const uint32_t have[2] = {c0, c1};
        __syncthreads();
        // the digit in which it is reached; where rounding leaves none, the last one that holds a token
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (!have[e]) continue;
            atomicMax(&s.at[2], d + e + 1);
            if (reached(in[e])) atomicMax(&s.at[1], kBins - (d + e));
        }
        __syncthreads();
        const int digit = s.at[1] ? kBins - s.at[1] : s.at[2] - 1;
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (d + e == digit) { s.sums[0] = out[e].mass; s.at[3] = (int)out[e].count; }
        __syncthreads();
        before = Prefix{s.sums[0], (uint32_t)s.at[3]};
        prefix |= (uint64_t)digit << shift;
        __syncthreads();
    }
    return prefix;
}

template <int DT>
__device__ __forceinline__ void resolve_many(SampleLds &s, uint64_t *hist_mass, uint32_t *hist_count, const SampleParams &p, int row, const RowRule &r,
                                             const Cuts &c) {
    auto weight = [&](uint64_t key) { return weight_of(exponent_of(key_logit(key), s.top, r)); };
    // sums up to and with a token, in order: what the k tokens hold, then where the kept ones end
    uint64_t all = s.mass[kBins - 1];
    uint32_t count = c.n;
    Prefix before;
    if (c.k_bin < kBins) {
        count = r.top_k;
        all = mass_before(s, c.k_bin);
        if (c.k_inside) {
            const uint64_t key = descend<DT>(s, hist_mass, hist_count, p, row, r, c.k_bin, before, [&](Prefix v) { return v.count >= r.top_k; });
            all = before.mass + weight(key);
        }
    }
    if (r.by_p) {                                          // the last token with less than the limit before it is the first to reach it
        const double limit = r.top_p * (double)all;
        const int b = first_bin(s, [&](int i) { return s.count[i] && (double)s.mass[i] >= limit; });
        const uint64_t key = descend<DT>(s, hist_mass, hist_count, p, row, r, b, before, [&](Prefix v) { return (double)v.mass >= limit; });
        if (before.count + 1 < count) { count = before.count + 1; all = before.mass + weight(key); }
    }
    if (r.by_min) {                                        // by value: its bin's tokens are added up in one pass
        const int b = bin_of(r.min_a);
        if (count_before(s, b) < count) {
            __syncthreads();
            if (threadIdx.x == 0) { s.sums[1] = mass_before(s, b); s.n_cand = count_before(s, b); }
            __syncthreads();
            const uint4 *base;
            int phase;
            const int pieces = row_pieces<DT>(p, row, base, phase);
            for_tokens<DT>(p, base, phase, 0, pieces, [&](uint32_t, float x) {
                const double a = exponent_of(x, s.top, r);
                if (bin_of(a) != b || a < r.min_a) return;
                atomicAdd((unsigned long long *)&s.sums[1], (unsigned long long)weight_of(a));
                atomicAdd(&s.n_cand, 1u);
            });
            __syncthreads();
            if (s.n_cand < count) { count = s.n_cand; all = s.sums[1]; }
            __syncthreads();
        }
    }
    const double target = r.u * (double)all;
    const int b = first_bin(s, [&](int i) { return (double)s.mass[i] > target; });
    const uint64_t key = descend<DT>(s, hist_mass, hist_count, p, row, r, b, before, [&](Prefix v) { return (double)v.mass > target; });
    if (threadIdx.x == 0) answer(p, row, key, s.top, r, all);
}

__device__ __forceinline__ float block_max(SampleLds &s, float top) {
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave_count[threadIdx.x >> 6] = __float_as_uint(top);
    __syncthreads();
    top = __uint_as_float(s.wave_count[threadIdx.x & 15]);
#pragma unroll
    for (int d = 8; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    return top;
}

__device__ __forceinline__ uint32_t needed_tokens(const SampleLds &s) {
    uint32_t n = 0;
    for (int q = 0; q < kBins / 32; q++)
        for (uint32_t bits = s.need[q]; bits; bits &= bits - 1) {
            const int b = 32 * q + __ffs((int)bits) - 1;
            n += s.count[b] - count_before(s, b);
        }
    return n;
}
template <int DT>
__device__ __forceinline__ void histogram(SampleLds &s, const SampleParams &p, const RowRule &r, const uint4 *base, int phase, int from, int to, float top) {
    for_tokens<DT>(p, base, phase, from, to, [&](uint32_t, float x) {
        const double a = exponent_of(x, top, r);
        const int b = bin_of(a);
        atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)weight_of(a));
        atomicAdd(&s.count[b], 1u);
    });
}
__device__ __forceinline__ void no_token(const SampleParams &p, int row) {
    p.token[row] = -1;
    if (p.logprob) p.logprob[row] = -INFINITY;
}

// ---- few rows: a row's slices on workgroups of their own, three launches ----
// What crosses workgroups inside a launch goes past the L2s (far_load, far_store, atomics); the last of a row's workgroups to get
// there goes on alone, none waits for another.
__device__ __forceinline__ bool last_to_arrive(SampleLds &s, uint32_t *counter) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // this wavefront's stores and atomics have reached memory
    __syncthreads();
    if (threadIdx.x == 0) s.at[0] = (int)atomicAdd(counter, 1u);
    __syncthreads();
    return s.at[0] == (int)gridDim.x - 1;
}
template <int DT> __device__ __forceinline__ void row_slice(const SampleParams &p, const uint4 *&base, int &phase, int &from, int &to) {
    const int pieces = row_pieces<DT>(p, blockIdx.y, base, phase), per = (pieces + (int)gridDim.x - 1) / (int)gridDim.x;
    from = min(per * (int)blockIdx.x, pieces);
    to = min(from + per, pieces);
}
template <int DT>
__global__ void __launch_bounds__(kSampThreads) slice_top_kernel(const SampleParams p, RowState *state) {
    __shared__ float tops[16];
    RowState &st = state[blockIdx.y];
    const uint4 *base;
    int phase, from, to;
    row_slice<DT>(p, base, phase, from, to);
    float top = -INFINITY;
    for_tokens<DT>(p, base, phase, from, to, [&](uint32_t, float x) { top = fmaxf(top, x); });
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    for (int i = (int)(blockIdx.x * kSampThreads + threadIdx.x); i < kBins; i += (int)gridDim.x * kSampThreads) { st.mass[i] = 0; st.count[i] = 0; }
    if (blockIdx.x == 0 && threadIdx.x < 4) (&st.n_need)[threadIdx.x] = 0;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; w++) top = fmaxf(top, tops[w]);
        st.slice_top[blockIdx.x] = top;
    }
}
__device__ __forceinline__ float slices_top(const RowState &st) {
    float top = -INFINITY;
    for (int i = 0; i < (int)gridDim.x; i++) top = fmaxf(top, st.slice_top[i]);
    return top;
}
template <int DT>
__global__ void __launch_bounds__(kSampThreads) slice_histogram_kernel(const SampleParams p, RowState *state) {
    extern __shared__ __align__(16) uint8_t lds[];
    SampleLds &s = *reinterpret_cast<SampleLds *>(lds);
    const int row = blockIdx.y;
    RowState &st = state[row];
    const float top = slices_top(st);
    if (top == -INFINITY) {
        if (blockIdx.x == 0 && threadIdx.x == 0) no_token(p, row);
        return;
    }
    const RowRule r = row_rule(p, row);
    for (int i = threadIdx.x; i < kBins; i += kSampThreads) { s.mass[i] = 0; s.count[i] = 0; }
    __syncthreads();
    const uint4 *base;
    int phase, from, to;
    row_slice<DT>(p, base, phase, from, to);
    histogram<DT>(s, p, r, base, phase, from, to, top);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kSampThreads)
        if (s.count[i]) {
            atomicAdd((unsigned long long *)&st.mass[i], (unsigned long long)s.mass[i]);
            atomicAdd(&st.count[i], s.count[i]);
        }
    if (!last_to_arrive(s, &st.arrived[0])) return;
    for (int i = threadIdx.x; i < kBins; i += kSampThreads) { s.mass[i] = far_load(&st.mass[i]); s.count[i] = far_load(&st.count[i]); }
    __syncthreads();
    scan_bins(s);
    mark_bins(s, r, find_cuts(s, r));
    for (int i = threadIdx.x; i < kBins; i += kSampThreads) { st.mass[i] = s.mass[i]; st.count[i] = s.count[i]; }      // (sums from here on)
    if (threadIdx.x < kBins / 32) st.need[threadIdx.x] = s.need[threadIdx.x];
    if (threadIdx.x == 0) st.n_need = needed_tokens(s);
}
template <int DT>
__global__ void __launch_bounds__(kSampThreads) slice_resolve_kernel(const SampleParams p, RowState *state) {
    extern __shared__ __align__(16) uint8_t lds[];
    SampleLds &s = *reinterpret_cast<SampleLds *>(lds);
    uint64_t *hist_mass = reinterpret_cast<uint64_t *>(lds + sizeof(SampleLds));
    const int row = blockIdx.y;
    RowState &st = state[row];
    const float top = slices_top(st);
    if (top == -INFINITY) return;
    const RowRule r = row_rule(p, row);
    const uint32_t n = st.n_need;
    if (threadIdx.x < kBins / 32) s.need[threadIdx.x] = st.need[threadIdx.x];
    if (threadIdx.x == 0) s.top = top;
    __syncthreads();
    if (n <= kCand) {
        const uint4 *base;
        int phase, from, to;
        row_slice<DT>(p, base, phase, from, to);
        for_tokens<DT>(p, base, phase, from, to, [&](uint32_t idx, float x) {
            if (needed(s, bin_of(exponent_of(x, top, r)))) far_store(&st.cand[min(atomicAdd(&st.n_cand, 1u), (uint32_t)kCand - 1u)], order_key(x, idx));
        });
        if (!last_to_arrive(s, &st.arrived[1])) return;
    } else if (blockIdx.x) {
        return;
    }
    for (int i = threadIdx.x; i < kBins; i += kSampThreads) { s.mass[i] = st.mass[i]; s.count[i] = st.count[i]; }
    if (n <= kCand)
        for (uint32_t i = threadIdx.x; i < n; i += kSampThreads) s.cand[i] = far_load(&st.cand[i]);
    __syncthreads();
    const Cuts c = find_cuts(s, r);
    if (n <= kCand) resolve_few(s, p, row, r, c, n);
    else resolve_many<DT>(s, hist_mass, reinterpret_cast<uint32_t *>(hist_mass + kBins), p, row, r, c);
}

// One workgroup a row.
template <int DT>
__global__ void __launch_bounds__(kSampThreads) sample_rows_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t lds[];
    SampleLds &s = *reinterpret_cast<SampleLds *>(lds);
    uint64_t *hist_mass = reinterpret_cast<uint64_t *>(lds + sizeof(SampleLds));
    uint32_t *hist_count = reinterpret_cast<uint32_t *>(hist_mass + kBins);
    const int row = blockIdx.x;
    const RowRule r = row_rule(p, row);
    const uint4 *base;
    int phase;
    const int pieces = row_pieces<DT>(p, row, base, phase);
    for (int i = threadIdx.x; i < kBins; i += kSampThreads) { s.mass[i] = 0; s.count[i] = 0; }
    float top = -INFINITY;
    for_tokens<DT>(p, base, phase, 0, pieces, [&](uint32_t, float x) { top = fmaxf(top, x); });
    top = block_max(s, top);
    if (top == -INFINITY) {                                // nothing can be chosen
        if (threadIdx.x == 0) no_token(p, row);
        return;
    }
    if (threadIdx.x == 0) { s.top = top; s.n_cand = 0; }
    __syncthreads();
    histogram<DT>(s, p, r, base, phase, 0, pieces, top);
    __syncthreads();
    scan_bins(s);
    const Cuts c = find_cuts(s, r);
    mark_bins(s, r, c);
    const uint32_t n = needed_tokens(s);
    if (n > kCand) {
        resolve_many<DT>(s, hist_mass, hist_count, p, row, r, c);
        return;
    }
    for_tokens<DT>(p, base, phase, 0, pieces, [&](uint32_t idx, float x) {
        if (needed(s, bin_of(exponent_of(x, top, r)))) s.cand[atomicAdd(&s.n_cand, 1u)] = order_key(x, idx);
    });
    __syncthreads();
    resolve_few(s, p, row, r, c, n);
}

// Slices a row: as many as make 256 workgroups, of 4096 logits or more; one where that leaves a single one.
static int sample_slices(const pkv_sample_args *a) {
    int g = (256 + a->rows - 1) / a->rows;
    g = g < a->vocab / 4096 ? g : a->vocab / 4096;
    return g < 1 ? 1 : g > kMaxSlices ? kMaxSlices : g;
}

static int sample_check(const pkv_sample_args *a) {
    PKV_REQUIRE(a != nullptr, PKV_ERR_INVALID, "null pointer argument");
    PKV_REQUIRE(a->dtype == PKV_F16 || a->dtype == PKV_BF16 || a->dtype == PKV_F32, PKV_ERR_UNSUPPORTED, "Unsupported data type");
    PKV_REQUIRE(a->rows > 0 && a->vocab > 0, PKV_ERR_INVALID, "sizes must be positive");
    PKV_REQUIRE(a->vocab <= (1 << 20), PKV_ERR_UNSUPPORTED, "not supported: %d tokens (at most 2^20)", a->vocab);
    return PKV_OK;
}

template <int DT> static int sample_launch(const SampleParams &p, int slices, void *workspace, hipStream_t s) {
    const size_t lds = sizeof(SampleLds) + kBins * 12;
    if (slices == 1) {
        PKV_HIP_CHECK(hipFuncSetAttribute((const void *)sample_rows_kernel<DT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        sample_rows_kernel<DT><<<dim3((unsigned)p.rows), kSampThreads, lds, s>>>(p);
    } else {
        RowState *state = (RowState *)workspace;
        const dim3 grid((unsigned)slices, (unsigned)p.rows);
        PKV_HIP_CHECK(hipFuncSetAttribute((const void *)slice_resolve_kernel<DT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        slice_top_kernel<DT><<<grid, kSampThreads, 0, s>>>(p, state);
        slice_histogram_kernel<DT><<<grid, kSampThreads, sizeof(SampleLds), s>>>(p, state);
        slice_resolve_kernel<DT><<<grid, kSampThreads, lds, s>>>(p, state);
    }
    PKV_HIP_CHECK(hipGetLastError());
    return PKV_OK;
}

}  // namespace pkv

extern "C" {

uint64_t pkv_sample_workspace(const pkv_sample_args *a) {
    using namespace pkv;
    if (sample_check(a)) return 0;
    return sample_slices(a) > 1 ? (uint64_t)a->rows * sizeof(RowState) : 0;
}

int pkv_sample(const pkv_sample_args *a, void *workspace, uint64_t workspace_bytes, pkv_stream_t s_) {
    using namespace pkv;
    hipStream_t s = (hipStream_t)s_;
    const int bad = sample_check(a);
    if (bad) return bad;
    PKV_REQUIRE(a->logits && a->u && a->token, PKV_ERR_INVALID, "null pointer argument");
    PKV_REQUIRE(a->row_stride >= 0 && reinterpret_cast<uintptr_t>(a->logits) % (a->dtype == PKV_F32 ? 4 : 2) == 0, PKV_ERR_INVALID,
                "bad row stride or address");
    static_assert(kF32 == PKV_F32, "data type codes");
    const int slices = sample_slices(a);
    const uint64_t need = pkv_sample_workspace(a);
    PKV_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0), PKV_ERR_CAPACITY,
                "the call needs a 16-byte aligned workspace of %llu bytes", (unsigned long long)need);
    SampleParams p;
    p.logits = a->logits; p.u = a->u; p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
    p.token = a->token; p.logprob = a->logprob; p.row_stride = a->row_stride; p.rows = a->rows; p.vocab = a->vocab;
    p.top_k_all = a->top_k_all; p.temperature_all = a->temperature_all; p.top_p_all = a->top_p_all; p.min_p_all = a->min_p_all;
    if (a->dtype == PKV_F16) return sample_launch<PKV_F16>(p, slices, workspace, s);
    if (a->dtype == PKV_BF16) return sample_launch<PKV_BF16>(p, slices, workspace, s);
    return sample_launch<kF32>(p, slices, workspace, s);
}

}  // extern "C"
