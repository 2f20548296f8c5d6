// A token for each row of logits from a given uniform number: temperature, top-k, top-p, min-p, and the draw.
//
// Order of a row: logit descending, equal logits by index.  Weight of a token: e = 2^-(y / 64), y = (max - logit) 64 log2(e) / T, its
// place.  Each filter keeps a prefix of the order -- the first k; the tokens with less than p of the k's mass before them; those with
// e >= min_p -- and the draw takes the first token whose inclusive mass exceeds u times the mass kept.  So nothing is sorted as a
// whole: a histogram over the whole parts of y (2816 bins, counts and masses) says in which bins a filter can end and in which the
// draw can fall; only those bins' tokens are gathered, ordered and looked at one by one.
//
// Exact whatever the order of the additions: weights are formed in fp64 and held as integers of 2^-43, their sums are whole numbers
// (below 2^63 for 2^20 tokens), so a row gives the same token from any number of workgroups.  Two tokens of a row of 150000 are told
// apart at 10^-13 of its mass, against 2^-24 of the uniform numbers.
//
// A row is read three times: its maximum, the histogram, the gathering.  Many rows are bound by the histogram's instructions and LDS
// atomics (vector units 53 % busy, LDS 28 %), not by bytes: 256 rows of 151936 in bf16 80 us, 69 with top-k 50, 91 with top-p 0.9 (more
// candidates), 88 with settings of every kind, where reading them once takes 15; held in registers between the passes the rows took 2 %
// less, not worth a second way of reading.  Few rows are bound by the latency of what follows one another: a row of 151936 20.5 us in three
// launches (3 + 12 + 6), a row of temperature 0 8.5 us.
#include "pkv_block.hpp"
#include "pkv_runtime.hpp"

namespace pkv {

constexpr int kSampThreads = 1024, kFracBits = 43;
constexpr double kPerUnit = 64.0;                          // bins for each halving of the weight
// Behind 44 halvings weights are below half of 2^-43: such tokens have no mass, so they are never drawn, and where a filter ends among
// them makes no difference.  The bins go a little further, to three a thread.
constexpr int kNoMass = 44 * 64, kMine = 3, kBins = kMine * kSampThreads, kCand = kBins;    // (kCand: tokens looked at one by one)
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
    double per_logit, top_p, last, u;                      // place y = (max - logit) * per_logit; min-p keeps y <= last
    uint32_t top_k;                                        // 0: off
    bool by_p, by_min;
};
__device__ __forceinline__ RowRule row_rule(const SampleParams &p, int row, float largest) {
    RowRule r;
    float t = p.temperature ? p.temperature[row] : p.temperature_all;
    const float top = p.top_p ? p.top_p[row] : p.top_p_all, least = p.min_p ? p.min_p[row] : p.min_p_all;
    const int k = p.top_k ? p.top_k[row] : p.top_k_all;
    r.top_k = k > 0 ? (uint32_t)k : 0u;
    if (!(t > 0.f)) { t = 1.f; r.top_k = 1; }              // temperature 0: the first of the order
    r.per_logit = largest == INFINITY ? kPerUnit : kPerUnit * 1.4426950408889634074 / (double)t;   // (behind +inf at any temperature)
    r.by_p = top < 1.f;
    r.top_p = fmax((double)top, 0.0);
    r.by_min = least > 0.f;
    r.last = r.by_min ? fmax(-kPerUnit * log2((double)least), 0.0) : 0.0;
    r.u = fmin(fmax((double)p.u[row], 0.0), 1.0 - 0x1p-30);
    return r;
}
__device__ __forceinline__ double place_of(float x, float top, const RowRule &r) {
    return fmax(((double)top - (double)x) * r.per_logit, 0.0);             // (inf - inf: 0)
}
__device__ __forceinline__ int bin_of(double y) { return (int)fmin(y, (double)(kBins - 1)); }
// 2^-(y / 64) as a whole number of 2^-43: base[bin] = 2^(43 - bin / 64), times the series of 2^-(f / 64) for what is left of the place,
// 0 <= f < 1, to the fifth power (the rest is below 2^-48).  Right for bins in front of kNoMass.
__device__ __forceinline__ uint64_t weight_of(const double *base, double y, int bin) {
    const double f = __builtin_amdgcn_fract(y);
    constexpr double c = 0.69314718055994530942 / kPerUnit;
    double e = -c * c * c * c * c / 120.0;
    e = fma(e, f, c * c * c * c / 24.0);
    e = fma(e, f, -c * c * c / 6.0);
    e = fma(e, f, c * c / 2.0);
    e = fma(e, f, -c);
    e = fma(e, f, 1.0);
    const double fixed = fma(e, base[bin], 0x1p52);        // (the low bits of the sum are the rounded number)
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

// A row in 16-byte pieces (piece 0 holds its first logit): the pieces are aligned, so the first and the last may hold others' bytes as
// well, which count as -inf.
template <int DT> __device__ __forceinline__ int row_pieces(const SampleParams &p, int row, const uint4 *&base, int &phase) {
    constexpr int ES = DT == kF32 ? 4 : 2;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.logits) + (uintptr_t)((int64_t)row * p.row_stride) * ES;
    base = reinterpret_cast<const uint4 *>(at & ~(uintptr_t)15);
    phase = (int)(at & 15) / ES;
    return (phase + p.vocab + 16 / ES - 1) / (16 / ES);
}
// f(index of the first, logits, the largest) for pieces from .. to - 1, called by whole wavefronts but for lanes that ran out.
template <int DT, int U = 4, class F>
__device__ __forceinline__ void for_pieces(const SampleParams &p, const uint4 *base, int phase, int from, int to, F f) {
    constexpr int N = DT == kF32 ? 4 : 8;                  // U pieces in flight a thread
    for (int c0 = from + (int)threadIdx.x; c0 < to; c0 += U * kSampThreads) {
        uint4 v[U];
#pragma unroll
        for (int i = 0; i < U; i++) v[i] = base[min(c0 + i * kSampThreads, to - 1)];
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int c = c0 + i * kSampThreads;
            if (c >= to) break;
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            float x[N];
#pragma unroll
            for (int e = 0; e < N; e++) {
                if (DT == kF32) x[e] = __uint_as_float(w[e]);
                else if (DT == PKV_F16) x[e] = __half2float(__ushort_as_half((unsigned short)(w[e >> 1] >> (16 * (e & 1)))));
                else x[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
            }
            const int idx = c * N - phase;
            if (idx < 0 || idx + N > p.vocab) {
#pragma unroll
                for (int e = 0; e < N; e++)
                    if ((uint32_t)(idx + e) >= (uint32_t)p.vocab) x[e] = -INFINITY;
            }
            float top = x[0];
#pragma unroll
            for (int e = 1; e < N; e++) top = fmaxf(top, x[e]);            // (NaN: the other one)
            f(idx, x, top);
        }
    }
}
template <int DT>
__device__ __forceinline__ float largest(const SampleParams &p, const uint4 *base, int phase, int from, int to) {
    float top = -INFINITY;
    for_pieces<DT>(p, base, phase, from, to, [&](int, const float *, float x) { top = fmaxf(top, x); });
    return top + 0.f;                                      // (-0 equals 0)
}
// f(index, logit) for the tokens with a logit of `least` (a finite number) or more; NaN has none.
template <int DT, class F>
__device__ __forceinline__ void for_tokens(const SampleParams &p, const uint4 *base, int phase, int from, int to, float least, F f) {
    constexpr int N = DT == kF32 ? 4 : 8;
    for_pieces<DT, 1>(p, base, phase, from, to, [&](int idx, const float *x, float top) {
        if (!__any(top >= least)) return;
#pragma unroll
        for (int e = 0; e < N; e++)
            if (x[e] >= least) f((uint32_t)(idx + e), x[e] + 0.f);
    });
}
// A finite logit below which every place is at `bin` or behind it, whatever the roundings: one fp32 comparison instead of the place.
__device__ __forceinline__ float surely_behind(float top, int bin, const RowRule &r) {
    const double x = (double)top - ((double)bin + 1.0) / r.per_logit;
    return fabs((double)top) < 3.0e38 && x > -3.0e38 ? (float)(x - fabs(x) * 0x1p-22) : -3.402823466e38f;
}

// A run of bins whose tokens are looked at one by one: what lies in front of it and in it.
struct Span {
    int from, to;                                          // (from > to: none)
    uint32_t count, size;
    uint64_t mass, total;
};
// What the histogram says about a row.
struct RowPlan {
    float top;
    uint32_t gathered;                                     // tokens in the spans
    uint64_t k_mass, low_mass;                             // mass of the k tokens unless the k-th is in a span; of what is kept for certain
    int k_inside, k_limits;                                // top-k ends inside a bin; anywhere
    Span span[3];
};
// What the launches of a split call hand on, in the workspace: one of these a row.
constexpr int kMaxSlices = 64;                             // (a lane each where they are put together)
struct RowState {
    uint64_t mass[kBins], cand[kCand];
    uint32_t count[kBins];
    float slice_top[kMaxSlices];
    RowPlan plan;
    uint32_t n_cand, arrived[2];
};
template <class T> __device__ __forceinline__ T far_load(const T *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class T> __device__ __forceinline__ void far_store(T *p, T x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct Prefix { uint64_t mass; uint32_t count; };

// What a row's resolution keeps in LDS.
struct SampleLds {
    uint64_t mass[kBins];                                  // of the bin; after scan_bins: up to and with it; then the candidates' weights
    uint64_t cand[kCand];                                  // keys; of a row resolved by digits the digits' masses and counts
    uint32_t count[kBins];
    uint64_t wave_mass[16];
    uint32_t wave_count[16];
    float edge[6];
    double base[kBins];                                    // weight of a bin's first place
    float top;
    uint32_t n_cand;
    uint64_t best, sums[2];
    int at[8];
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
#pragma unroll 5
    for (int w = 0; w < kSampThreads / 64 - 1; w++) {      // (five are read at once)
        const uint64_t m = s.wave_mass[w];
        const uint32_t c = s.wave_count[w];
        v.mass += w < wave ? m : 0ull;
        v.count += w < wave ? c : 0u;
    }
    return v;
}
// A thread's own bins' inclusive sums; [0]: what lies in front of them.
struct MyBins { uint64_t mass[kMine + 1]; uint32_t count[kMine + 1]; };
// The histogram, load(bin, mass, count), becomes inclusive sums in s.mass and s.count, and at[] is made ready for the searches.
template <class F> __device__ __forceinline__ MyBins scan_bins(SampleLds &s, F load) {
    const int b = kMine * threadIdx.x;
    MyBins r;
    r.mass[0] = 0;
    r.count[0] = 0;
#pragma unroll
    for (int i = 0; i < kMine; i++) load(b + i, r.mass[i + 1], r.count[i + 1]);
#pragma unroll
    for (int i = 0; i < kMine; i++) { r.mass[i + 1] += r.mass[i]; r.count[i + 1] += r.count[i]; }
    const Prefix v = block_scan(s, Prefix{r.mass[kMine], r.count[kMine]});
    const uint64_t m0 = v.mass - r.mass[kMine];
    const uint32_t c0 = v.count - r.count[kMine];
#pragma unroll
    for (int i = 0; i <= kMine; i++) { r.mass[i] += m0; r.count[i] += c0; }
#pragma unroll
    for (int i = 0; i < kMine; i++) { s.mass[b + i] = r.mass[i + 1]; s.count[b + i] = r.count[i + 1]; }
    if (threadIdx.x < 8) s.at[threadIdx.x] = kBins;
    __syncthreads();
    return r;
}
// at[slot] = the first bin whose inclusive sums satisfy the condition, out of registers; there behind the next barrier.
template <class F> __device__ __forceinline__ void search_mine(SampleLds &s, int slot, const MyBins &mine, F holds) {
    if (!holds(mine.mass[kMine], mine.count[kMine]) || (threadIdx.x && holds(mine.mass[0], mine.count[0]))) return;
#pragma unroll
    for (int i = kMine - 1; i >= 0; i--)
        if (holds(mine.mass[i + 1], mine.count[i + 1])) s.at[slot] = kMine * threadIdx.x + i;
}
// at[slot] = the first bin whose inclusive sum satisfies the condition (kBins: none); there behind the next barrier.
template <class F> __device__ __forceinline__ void search_bin(SampleLds &s, int slot, F holds) {
    const int b = kMine * threadIdx.x;
    if (!holds(b + kMine - 1) || (b && holds(b - 1))) return;
#pragma unroll
    for (int i = kMine - 1; i >= 0; i--)
        if (holds(b + i)) s.at[slot] = b + i;
}
template <class F> __device__ __forceinline__ int first_bin(SampleLds &s, F holds) {
    __syncthreads();
    if (threadIdx.x == 0) s.at[7] = kBins;
    __syncthreads();
    search_bin(s, 7, holds);
    __syncthreads();
    return s.at[7];
}
__device__ __forceinline__ uint64_t mass_before(const SampleLds &s, int bin) { return bin ? s.mass[bin - 1] : 0ull; }
__device__ __forceinline__ uint32_t count_before(const SampleLds &s, int bin) { return bin ? s.count[bin - 1] : 0u; }

__device__ __forceinline__ void order_spans(Span &a, Span &b) {            // the earlier one first; overlapping ones become one
    if (b.from > b.to) return;
    if (a.from > a.to || b.from < a.from) { const Span t = a; a = b; b = t; }
    if (b.from > b.to || b.from > a.to + 1) return;
    a.to = max(a.to, b.to);
    b.from = 1; b.to = 0;
}
// Which bins the answer depends on one by one, from the scanned histogram: the one that the k-th token is in, those in which the last
// kept token can be, those in which the draw can fall.  The same in every thread.
__device__ __forceinline__ RowPlan make_plan(SampleLds &s, const MyBins &mine, const RowRule &r, float top) {
    RowPlan p;
    p.top = top;
    const uint64_t all = s.mass[kBins - 1];
    int k_bin = kBins;                                     // top-k ends inside this bin, or in front of it
    p.k_inside = 0;
    p.k_limits = r.top_k && r.top_k < s.count[kBins - 1];  // (of the tokens that have mass)
    uint64_t k_low = all, k_high = all;                    // mass of the k tokens, between these
    if (p.k_limits) {
        search_mine(s, 0, mine, [&](uint64_t, uint32_t c) { return c >= r.top_k; });
        __syncthreads();
        const int b = s.at[0];
        p.k_inside = s.count[b] != r.top_k;
        k_bin = p.k_inside ? b : b + 1;
        k_low = p.k_inside ? mass_before(s, b) : s.mass[b];
        k_high = s.mass[b];
    }
    p.k_mass = k_low;
    int low = k_bin, high = k_bin;                         // the bins in which the last kept token can be (kBins: all are kept)
    if (r.by_p) {
        const double from = r.top_p * (double)k_low, to = r.top_p * (double)k_high;
        search_mine(s, 1, mine, [&](uint64_t m, uint32_t c) { return c && (double)m >= from; });
        search_mine(s, 2, mine, [&](uint64_t m, uint32_t c) { return c && (double)m >= to; });
        __syncthreads();
        low = min(low, s.at[1]);
        high = min(high, s.at[2]);
    }
    const bool by_min = r.by_min && bin_of(r.last) < kNoMass;
    if (by_min) {
        low = min(low, bin_of(r.last));
        high = min(high, bin_of(r.last));
    }
    p.low_mass = low < kBins ? mass_before(s, low) : all;
    const bool whole = high >= kBins || (high == k_bin && !p.k_inside);    // the last bin that can hold a kept token is kept as a whole
    const uint64_t high_mass = high >= kBins ? all : whole ? mass_before(s, high) : s.mass[high];
    const double from = r.u * (double)max(p.low_mass, (1ull << kFracBits) - 1ull), to = r.u * (double)max(high_mass, 1ull << kFracBits);
    search_mine(s, 3, mine, [&](uint64_t m, uint32_t) { return (double)m > from; });
    search_mine(s, 4, mine, [&](uint64_t m, uint32_t) { return (double)m > to; });
    __syncthreads();
    p.span[0].from = k_bin; p.span[0].to = p.k_inside ? k_bin : -1;
    p.span[1].from = low; p.span[1].to = r.by_p || by_min ? min(whole ? high - 1 : high, kBins - 1) : -1;
    p.span[2].from = s.at[3]; p.span[2].to = min(s.at[4], kBins - 1);
    order_spans(p.span[0], p.span[1]);
    order_spans(p.span[1], p.span[2]);
    order_spans(p.span[0], p.span[1]);
    order_spans(p.span[1], p.span[2]);
    p.gathered = 0;
#pragma unroll
    for (int i = 0; i < 3; i++) {
        Span &v = p.span[i];
        const bool is = v.from <= v.to;
        v.count = is ? count_before(s, v.from) : 0u;
        v.mass = is ? mass_before(s, v.from) : 0ull;
        v.size = is ? s.count[v.to] - v.count : 0u;
        v.total = is ? s.mass[v.to] - v.mass : 0ull;
        p.gathered += v.size;
    }
    return p;
}

// The value of lane ^ J, without LDS.
template <int J> __device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if (J == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);             // (quads 1 0 3 2)
    if (J == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);             // (2 3 0 1)
    if (J == 4) return (uint32_t)__builtin_amdgcn_update_dpp(0, __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true), 0x1B, 0xF, 0xF, true);   // (7 - i, then 3 - i)
    if (J == 8) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true);            // (rows of 16 turned by 8)
    if (J == 16) {
        const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? both[0] : both[1];
    }
    const auto both = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? both[0] : both[1];
}
template <int J> __device__ __forceinline__ uint64_t lane_xor64(uint64_t v) {
    return ((uint64_t)lane_xor<J>((uint32_t)(v >> 32)) << 32) | lane_xor<J>((uint32_t)v);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
    v = max(v, lane_xor64<1>(v));
    v = max(v, lane_xor64<2>(v));
    v = max(v, lane_xor64<4>(v));
    v = max(v, lane_xor64<8>(v));
    v = max(v, lane_xor64<16>(v));
    return max(v, lane_xor64<32>(v));
}
// A wavefront's 64 keys in ascending order.
template <int K, int J> __device__ __forceinline__ void sort_step(uint64_t &key) {
    const int lane = threadIdx.x & 63;
    const uint64_t other = lane_xor64<J>(key);
    const bool low = ((lane & J) == 0) == ((lane & K) == 0);
    key = (other < key) == low ? other : key;
    if constexpr (J > 1) sort_step<K, J / 2>(key);
}
__device__ __forceinline__ uint64_t sort_wave(uint64_t key) {
    sort_step<2, 1>(key);
    sort_step<4, 2>(key);
    sort_step<8, 4>(key);
    sort_step<16, 8>(key);
    sort_step<32, 16>(key);
    sort_step<64, 32>(key);
    return key;
}
// The keys s.cand[0 .. n) in ascending order, there or in s.mass.  A wavefront sorts 64 in registers; then runs are merged in pairs, a
// key's place being its own in its run plus how many of the other run are smaller, which a search finds: a barrier for each doubling,
// where a sort across the workgroup has one for each of its steps (512 keys: 3 against 45).
__device__ __forceinline__ const uint64_t *sort_candidates(SampleLds &s, uint32_t n) {
    const int lane = threadIdx.x & 63;
    const uint32_t chunks = (n + 63) / 64, all = 64 * chunks;
    for (uint32_t c = threadIdx.x >> 6; c < chunks; c += kSampThreads / 64) {
        const uint64_t key = sort_wave(64 * c + lane < n ? s.cand[64 * c + lane] : ~0ull);
        s.cand[64 * c + lane] = key;
    }
    __syncthreads();
    uint64_t *from = s.cand, *to = s.mass;
    for (uint32_t run = 64; run < all; run *= 2) {
        for (uint32_t i = threadIdx.x; i < all; i += kSampThreads) {
            const uint64_t key = from[i];
            const uint32_t own = i & ~(run - 1u), other = own ^ run;
            uint32_t less = 0;
            if (other < all) {                             // (the last run may be shorter, or have no other)
                const uint32_t len = min(run, all - other);
                for (uint32_t step = run / 2; step; step >>= 1)
                    if (less + step <= len && from[other + less + step - 1] < key) less += step;
                if (less < len && from[other + less] < key) less++;
            }
            to[min(own, other) + (i - own) + less] = key;
        }
        __syncthreads();
        uint64_t *const t = from;
        from = to;
        to = t;
    }
    return from;
}

__device__ __forceinline__ void answer(const SampleParams &p, int row, uint64_t key, float top, const RowRule &r, uint64_t kept) {
    p.token[row] = (int64_t)(uint32_t)key;
    if (p.logprob) p.logprob[row] = (float)((-place_of(key_logit(key), top, r) / kPerUnit - (log2((double)kept) - kFracBits)) * 0.69314718055994530942);
}

// The answer from at most kCand gathered tokens (s.cand, behind a barrier; s.mass is not looked at any more).  All tokens of a span are
// there, so a candidate's rank and the mass in front of it are its span's plus those of the candidates of its span in front of it.
__device__ __forceinline__ void resolve_few(SampleLds &s, const SampleParams &p, int row, const RowRule &r, const RowPlan &plan) {
    const uint32_t n = plan.gathered;
    if (n <= 64) {                                         // one wavefront, a candidate a lane
        if (threadIdx.x >= 64) return;
        const int lane = threadIdx.x;
        const bool here = (uint32_t)lane < n;
        const uint64_t key = sort_wave(here ? s.cand[lane] : ~0ull);
        const double y = here ? place_of(key_logit(key), plan.top, r) : 0.0;
        const int bin = bin_of(y);
        const uint64_t w = here ? weight_of(s.base, y, bin) : 0ull;
        uint64_t sum = w;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t m = shfl_up64(sum, d);
            if (lane >= d) sum += m;
        }
        const Span &a = plan.span[0], &b = plan.span[1], &c = plan.span[2];
        const bool in_a = a.from <= a.to && bin <= a.to, in_b = !in_a && b.from <= b.to && bin <= b.to;
        const uint32_t rank = (uint32_t)lane + (in_a ? a.count : in_b ? b.count - a.size : c.count - a.size - b.size);
        const uint64_t upto = sum + (in_a ? a.mass : in_b ? b.mass - a.total : c.mass - a.total - b.total), front = upto - w;
        uint64_t k_mass = plan.k_mass;
        if (plan.k_inside) k_mass = max(k_mass, wave_max(here && rank + 1 == r.top_k ? upto : 0ull));
        const bool kept = here && (!plan.k_limits || rank < r.top_k) && (!r.by_p || rank == 0 || (double)front < r.top_p * (double)k_mass) &&
                          (!r.by_min || y <= r.last);
        const uint64_t total = max(plan.low_mass, wave_max(kept ? upto : 0ull));
        const uint64_t hit = __ballot(kept && (double)upto > r.u * (double)total);
        if (lane == (hit ? __ffsll((unsigned long long)hit) - 1 : 0)) answer(p, row, key, plan.top, r, total);
        return;
    }
    uint64_t key[kMine], w[kMine], front[kMine];
    int bin[kMine];
    double y[kMine];
    const uint64_t *sorted = sort_candidates(s, n);
#pragma unroll
    for (int e = 0; e < kMine; e++) {
        const uint32_t i = kMine * threadIdx.x + e;
        key[e] = ~0ull; w[e] = 0; y[e] = 0; bin[e] = 0;
        if (i < n) {
            key[e] = sorted[i];
            y[e] = place_of(key_logit(key[e]), plan.top, r);
            bin[e] = bin_of(y[e]);
            w[e] = weight_of(s.base, y[e], bin[e]);
        }
    }
    if (threadIdx.x == 0) { s.sums[0] = plan.k_mass; s.sums[1] = plan.low_mass; s.best = ~0ull; }
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < kMine; e++) { front[e] = sum; sum += w[e]; }
    const uint64_t ahead = block_scan(s, Prefix{sum, 0u}).mass - sum;
    uint32_t rank[kMine];
#pragma unroll
    for (int e = 0; e < kMine; e++) {
        const Span &a = plan.span[0], &b = plan.span[1], &c = plan.span[2];
        const bool in_a = a.from <= a.to && bin[e] <= a.to, in_b = !in_a && b.from <= b.to && bin[e] <= b.to;
        rank[e] = kMine * threadIdx.x + e + (in_a ? a.count : in_b ? b.count - a.size : c.count - a.size - b.size);
        front[e] += ahead + (in_a ? a.mass : in_b ? b.mass - a.total : c.mass - a.total - b.total);
        if (kMine * threadIdx.x + e < n && plan.k_inside && rank[e] + 1 == r.top_k) s.sums[0] = front[e] + w[e];
    }
    __syncthreads();
    const double limit = r.by_p ? r.top_p * (double)s.sums[0] : 0.0;
    // The order's sums rise, so of a wavefront's candidates the largest sum of a kept one, and the smallest key that reaches the target,
    // go on (an LDS atomic a candidate at one address, which the compiler makes a loop over the lanes, took 12 us for 140 of them).
    bool kept[kMine];
    uint64_t most = 0;
#pragma unroll
    for (int e = 0; e < kMine; e++) {
        kept[e] = kMine * threadIdx.x + e < n && (!plan.k_limits || rank[e] < r.top_k) && (!r.by_p || rank[e] == 0 || (double)front[e] < limit) &&
                  (!r.by_min || y[e] <= r.last);
        if (kept[e]) most = front[e] + w[e];
    }
    const bool any = kMine * (threadIdx.x & ~63u) < n;     // (uniform)
    if (any) {
        most = wave_max(most);
        if ((threadIdx.x & 63) == 0) atomicMax((unsigned long long *)&s.sums[1], (unsigned long long)most);
    }
    __syncthreads();
    const uint64_t total = s.sums[1];
    const double target = r.u * (double)total;
    if (any) {
        uint64_t best = ~0ull;
#pragma unroll
        for (int e = kMine - 1; e >= 0; e--)
            if (kept[e] && (double)(front[e] + w[e]) > target) best = key[e];
        best = ~wave_max(~best);
        if ((threadIdx.x & 63) == 0) atomicMin((unsigned long long *)&s.best, (unsigned long long)best);
    }
    __syncthreads();
    if (threadIdx.x == 0) answer(p, row, s.best, plan.top, r, total);
}

// ---- the answer when the bins in question hold more tokens than that (long runs of equal logits): by digits of the order ----
// The token at which a sum of the order first reaches what is asked for, among those of one bin: five passes over the row, each a
// histogram of the next digit (11 + 11 + 10 bits of the logit, 10 + 10 of the index) of the tokens that share the digits so far.
template <int DT, class F>
__device__ __forceinline__ uint64_t descend(SampleLds &s, const SampleParams &p, int row, const RowRule &r, int bin, Prefix &before, F reached) {
    constexpr int kDigits = 2048;
    uint64_t *hist_mass = s.cand;
    uint32_t *hist_count = reinterpret_cast<uint32_t *>(s.cand + kDigits);
    static_assert(kDigits * 12 <= sizeof(s.cand) && kDigits == 2 * kSampThreads, "two digits a thread, in the candidates' place");
    const uint4 *base;
    int phase;
    const int pieces = row_pieces<DT>(p, row, base, phase);
    uint64_t prefix = 0;
    before = Prefix{mass_before(s, bin), count_before(s, bin)};
    constexpr int kShift[5] = {53, 42, 32, 10, 0}, kWidth[5] = {11, 11, 10, 10, 10};
    for (int level = 0; level < 5; level++) {
        const int shift = kShift[level], above = shift + kWidth[level];
        __syncthreads();
        for (int i = threadIdx.x; i < kDigits; i += kSampThreads) { hist_mass[i] = 0; hist_count[i] = 0; }
        if (threadIdx.x == 0) { s.at[1] = 0; s.at[2] = 0; }
        __syncthreads();
        for_tokens<DT>(p, base, phase, 0, pieces, surely_behind(s.top, bin + 1, r), [&](uint32_t idx, float x) {
            const double y = place_of(x, s.top, r);
            if (bin_of(y) != bin) return;
            const uint64_t key = order_key(x, idx);
            if (above < 64 && (key >> above) != (prefix >> above)) return;
            const int digit = (int)((key >> shift) & ((1u << kWidth[level]) - 1u));
            atomicAdd((unsigned long long *)&hist_mass[digit], (unsigned long long)weight_of(s.base, y, bin));
            atomicAdd(&hist_count[digit], 1u);
        });
        __syncthreads();
        const int d = 2 * threadIdx.x;
        const uint64_t m0 = hist_mass[d], m1 = hist_mass[d + 1];
        const uint32_t c0 = hist_count[d], c1 = hist_count[d + 1];
        const Prefix v = block_scan(s, Prefix{m0 + m1, c0 + c1});
        const Prefix in[2] = {{before.mass + v.mass - m1, before.count + v.count - c1}, {before.mass + v.mass, before.count + v.count}};
        const Prefix out[2] = {{in[0].mass - m0, in[0].count - c0}, {in[1].mass - m1, in[1].count - c1}};
        const uint32_t have[2] = {c0, c1};
        // the digit in which it is reached; where rounding leaves none, the last one that holds a token
        int top = 0, last = 0;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (!have[e]) continue;
            last = d + e + 1;
            if (reached(in[e])) top = max(top, kDigits - (d + e));
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            top = max(top, __shfl_xor(top, o, 64));
            last = max(last, __shfl_xor(last, o, 64));
        }
        if ((threadIdx.x & 63) == 0) {
            atomicMax(&s.at[1], top);
            atomicMax(&s.at[2], last);
        }
        __syncthreads();
        const int digit = s.at[1] ? kDigits - s.at[1] : s.at[2] - 1;
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (d + e == digit) { s.sums[0] = out[e].mass; s.at[3] = (int)out[e].count; }
        __syncthreads();
        before = Prefix{s.sums[0], (uint32_t)s.at[3]};
        prefix |= (uint64_t)digit << shift;
    }
    __syncthreads();
    return prefix;
}

// (s.mass and s.count hold the sums.)
template <int DT>
__device__ __forceinline__ void resolve_many(SampleLds &s, const SampleParams &p, int row, const RowRule &r, const RowPlan &plan) {
    auto weight = [&](uint64_t key) {
        const double y = place_of(key_logit(key), s.top, r);
        return weight_of(s.base, y, bin_of(y));
    };
    // sums up to and with a token, in order: what the k tokens hold, then where the kept ones end
    uint64_t all = plan.k_mass;
    uint32_t count = plan.k_limits ? r.top_k : s.count[kBins - 1];
    Prefix before;
    if (plan.k_inside) {
        const int b = first_bin(s, [&](int i) { return s.count[i] >= r.top_k; });
        const uint64_t key = descend<DT>(s, p, row, r, b, before, [&](Prefix v) { return v.count >= r.top_k; });
        all = before.mass + weight(key);
    }
    if (r.by_p) {                                          // the last token with less than the limit before it is the first to reach it
        const double limit = r.top_p * (double)all;
        const int b = first_bin(s, [&](int i) { return s.count[i] && (double)s.mass[i] >= limit; });
        const uint64_t key = descend<DT>(s, p, row, r, b, before, [&](Prefix v) { return (double)v.mass >= limit; });
        if (before.count + 1 < count) { count = before.count + 1; all = before.mass + weight(key); }
    }
    if (r.by_min) {                                        // by value: its bin's tokens are added up in one pass
        const int b = bin_of(r.last);
        if (b < kNoMass && count_before(s, b) < count) {
            __syncthreads();
            if (threadIdx.x == 0) { s.sums[1] = mass_before(s, b); s.n_cand = count_before(s, b); }
            __syncthreads();
            const uint4 *base;
            int phase;
            const int pieces = row_pieces<DT>(p, row, base, phase);
            uint64_t sum = 0;
            uint32_t here = 0;
            for_tokens<DT>(p, base, phase, 0, pieces, surely_behind(s.top, b + 1, r), [&](uint32_t, float x) {
                const double y = place_of(x, s.top, r);
                if (bin_of(y) != b || y > r.last) return;
                sum += weight_of(s.base, y, b);
                here++;
            });
#pragma unroll
            for (int d = 32; d; d >>= 1) {
                sum += ((uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)(sum >> 32), d, 64) << 32) + (uint32_t)__shfl_xor((int)(uint32_t)sum, d, 64);
                here += (uint32_t)__shfl_xor((int)here, d, 64);
            }
            if ((threadIdx.x & 63) == 0) {
                atomicAdd((unsigned long long *)&s.sums[1], (unsigned long long)sum);
                atomicAdd(&s.n_cand, here);
            }
            __syncthreads();
            if (s.n_cand < count) { count = s.n_cand; all = s.sums[1]; }
            __syncthreads();
        }
    }
    const double target = r.u * (double)all;
    const int b = first_bin(s, [&](int i) { return (double)s.mass[i] > target; });
    const uint64_t key = descend<DT>(s, p, row, r, b, before, [&](Prefix v) { return (double)v.mass > target; });
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

// Counts and masses by bin, of the tokens that have mass, into s.mass and s.count.
template <int DT>
__device__ __forceinline__ void histogram(SampleLds &s, const SampleParams &p, const RowRule &r, const uint4 *base, int phase, int from, int to, float top) {
    for (int i = threadIdx.x; i < kBins; i += kSampThreads) { s.mass[i] = 0; s.count[i] = 0; }
    __syncthreads();
    const float least = surely_behind(top, kNoMass, r);
    for_pieces<DT>(p, base, phase, from, to, [&](int, const float *x, float most) {
        if (!__any(most >= least)) return;
        // four at a time without a branch: one token's steps wait for each other, four tokens' do not
#pragma unroll
        for (int e0 = 0; e0 < (DT == kF32 ? 4 : 8); e0 += 4) {
            uint64_t w[4];
            int b[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double y = place_of(x[e0 + e], top, r);
                b[e] = bin_of(y);
                w[e] = weight_of(s.base, y, b[e]);
            }
            asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));                     // (not one by one behind the tests below)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (x[e0 + e] >= least && b[e] < kNoMass) {
                    atomicAdd((unsigned long long *)&s.mass[b[e]], (unsigned long long)w[e]);
                    atomicAdd(&s.count[b[e]], 1u);
                }
        }
    });
    __syncthreads();
}
// The smallest logit with its place in `bin` or in front of it (the place falls with the logit, so there is one), by a wavefront: of the
// 64 numbers around where it should be the first one that is; near 0 beside a large maximum these are too close together, and a search
// finds it.
__device__ __forceinline__ float least_of(float top, int bin, const RowRule &r) {
    const auto ordered = [](float x) { const int b = (int)__float_as_uint(x); return b < 0 ? b ^ 0x7FFFFFFF : b; };
    const auto number = [](int b) { return __uint_as_float((uint32_t)(b < 0 ? b ^ 0x7FFFFFFF : b)); };
    const auto holds = [&](int b) { return bin_of(place_of(number(b), top, r)) <= bin; };
    int from = ordered(-3.402823466e38f), to = ordered(top);
    const double x = (double)top - ((double)bin + 1.0) / r.per_logit;
    const int near = ordered((float)fmin(fmax(x, -3.0e38), 3.0e38)) - 32, mine = min(max(near + (int)(threadIdx.x & 63), from), to);
    const uint64_t ok = __ballot(holds(mine));
    if (ok && !(ok & 1ull)) return number(__builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)ok) - 1));
    while (from < to) {
        const int mid = (int)(((int64_t)from + to) >> 1);
        if (holds(mid)) to = mid;
        else from = mid + 1;
    }
    return number(to);
}
// Tokens of the spans: reserve(how many) -> the first's number, for a wavefront's of a piece, then put(number, key) for each.  Two fp32
// comparisons a token and span with the spans' exact ends; a span that is not there lets none through.
template <int DT, class R, class F>
__device__ __forceinline__ void gather(SampleLds &s, const SampleParams &p, const RowRule &r, const RowPlan &plan, const uint4 *base, int phase, int from, int to,
                                       R reserve, F put) {
    constexpr int N = DT == kF32 ? 4 : 8;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    int first[3], last[3];
#pragma unroll
    for (int i = 0; i < 3; i++) { first[i] = plan.span[i].from; last[i] = plan.span[i].to; }
    if (wave < 6) {
        const bool above = wave >= 3;
        const int f = wave % 3 == 0 ? first[0] : wave % 3 == 1 ? first[1] : first[2], l = wave % 3 == 0 ? last[0] : wave % 3 == 1 ? last[1] : last[2];
        float edge = above ? NAN : INFINITY;
        if (f <= l && !(above && f == 0)) edge = least_of(plan.top, above ? f - 1 : l, r);
        s.edge[wave] = edge;
    }
    __syncthreads();
    float low[3], above[3];                                // in a span: low <= x and not above <= x
#pragma unroll
    for (int i = 0; i < 3; i++) { low[i] = s.edge[i]; above[i] = s.edge[3 + i]; }
    const float least = fminf(fminf(low[0], low[1]), low[2]);
    const bool more = first[1] <= last[1];                // (the first is always there, and absent ones are last)
    for_pieces<DT, 2>(p, base, phase, from, to, [&](int idx, const float *x, float most) {
        if (!__any(most >= least)) return;
        uint64_t in[N];
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < N; e++) in[e] = __ballot((x[e] >= low[0]) & !(x[e] >= above[0]));
        if (more) {
#pragma unroll
            for (int e = 0; e < N; e++) in[e] |= __ballot(((x[e] >= low[1]) & !(x[e] >= above[1])) | ((x[e] >= low[2]) & !(x[e] >= above[2])));
        }
#pragma unroll
        for (int e = 0; e < N; e++) n += (uint32_t)__popcll(in[e]);
        if (!n) return;
        uint32_t at = reserve(n);
#pragma unroll
        for (int e = 0; e < N; e++) {
            if ((in[e] >> (threadIdx.x & 63)) & 1ull) put(at + __builtin_amdgcn_mbcnt_hi((uint32_t)(in[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], 0u)), order_key(x[e] + 0.f, (uint32_t)(idx + e)));
            at += (uint32_t)__popcll(in[e]);
        }
    });
}
// A wavefront's share of a counter (its first lane is there).
__device__ __forceinline__ uint32_t take(uint32_t *counter, uint32_t n) {
    uint32_t at = 0;
    if ((threadIdx.x & 63) == 0) at = atomicAdd(counter, n);
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
}
// top_k = 1 (temperature 0) needs no weights: the first token with the largest logit.  ~index, 0 where the pieces hold none, in every
// thread.
template <int DT>
__device__ __forceinline__ uint32_t first_largest(SampleLds &s, const SampleParams &p, const uint4 *base, int phase, int from, int to, float top) {
    uint32_t best = 0;
    for_pieces<DT>(p, base, phase, from, to, [&](int idx, const float *x, float most) {
        if (!__any(most >= top)) return;
#pragma unroll
        for (int e = 0; e < (DT == kF32 ? 4 : 8); e++)
            if (x[e] == top) best = max(best, ~(uint32_t)(idx + e));
    });
#pragma unroll
    for (int d = 32; d; d >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, d, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave_count[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < 16; w++) best = max(best, s.wave_count[w]);
    return best;
}
__device__ __forceinline__ void only_token(const SampleParams &p, int row, uint32_t best) {
    p.token[row] = (int64_t)~best;
    if (p.logprob) p.logprob[row] = 0.f;
}
__device__ __forceinline__ void fill_base(SampleLds &s) {
    static_assert(kSampThreads % 64 == 0, "a thread's bins are whole halvings apart");
    const double first = exp2((double)kFracBits - (double)(threadIdx.x & 63) / kPerUnit);
#pragma unroll
    for (int i = 0; i < kMine; i++) s.base[threadIdx.x + i * kSampThreads] = ldexp(first, -(int)((threadIdx.x + i * kSampThreads) >> 6));
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
    float top = largest<DT>(p, base, phase, from, to);
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    for (int i = (int)(blockIdx.x * kSampThreads + threadIdx.x); i < kBins; i += (int)gridDim.x * kSampThreads) { st.mass[i] = 0; st.count[i] = 0; }
    if (blockIdx.x == 0 && threadIdx.x == 0) st.n_cand = st.arrived[0] = st.arrived[1] = 0;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; w++) top = fmaxf(top, tops[w]);
        st.slice_top[blockIdx.x] = top;
    }
}
__device__ __forceinline__ float slices_top(const RowState &st) {
    const int lane = threadIdx.x & 63;
    float top = lane < (int)gridDim.x ? st.slice_top[lane] : -INFINITY;
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(top)));
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
    const RowRule r = row_rule(p, row, top);
    const uint4 *base;
    int phase, from, to;
    row_slice<DT>(p, base, phase, from, to);
    if (r.top_k == 1) {
        const uint32_t best = first_largest<DT>(s, p, base, phase, from, to, top);
        if (threadIdx.x == 0 && best) atomicMax(&st.n_cand, best);
        if (last_to_arrive(s, &st.arrived[0]) && threadIdx.x == 0) only_token(p, row, far_load(&st.n_cand));
        return;
    }
    fill_base(s);
    histogram<DT>(s, p, r, base, phase, from, to, top);
    for (int i = threadIdx.x; i < kBins; i += kSampThreads)
        if (s.count[i]) {
            atomicAdd((unsigned long long *)&st.mass[i], (unsigned long long)s.mass[i]);
            atomicAdd(&st.count[i], s.count[i]);
        }
    if (!last_to_arrive(s, &st.arrived[0])) return;
    const MyBins mine = scan_bins(s, [&](int i, uint64_t &m, uint32_t &c) { m = far_load(&st.mass[i]); c = far_load(&st.count[i]); });
    const RowPlan plan = make_plan(s, mine, r, top);
    if (threadIdx.x == 0) st.plan = plan;
    if (plan.gathered > kCand)                             // (sums from here on)
        for (int i = threadIdx.x; i < kBins; i += kSampThreads) { st.mass[i] = s.mass[i]; st.count[i] = s.count[i]; }
}
template <int DT>
__global__ void __launch_bounds__(kSampThreads) slice_resolve_kernel(const SampleParams p, RowState *state) {
    extern __shared__ __align__(16) uint8_t lds[];
    SampleLds &s = *reinterpret_cast<SampleLds *>(lds);
    const int row = blockIdx.y;
    RowState &st = state[row];
    const float top = slices_top(st);
    if (top == -INFINITY) return;
    const RowRule r = row_rule(p, row, top);
    if (r.top_k == 1) return;
    const RowPlan plan = st.plan;
    const uint32_t n = plan.gathered;
    fill_base(s);
    if (n > kCand) {
        if (blockIdx.x) return;
        for (int i = threadIdx.x; i < kBins; i += kSampThreads) { s.mass[i] = st.mass[i]; s.count[i] = st.count[i]; }
        if (threadIdx.x == 0) s.top = plan.top;
        __syncthreads();
        resolve_many<DT>(s, p, row, r, plan);
        return;
    }
    const uint4 *base;
    int phase, from, to;
    row_slice<DT>(p, base, phase, from, to);
    gather<DT>(s, p, r, plan, base, phase, from, to, [&](uint32_t n) { return take(&st.n_cand, n); },
               [&](uint32_t at, uint64_t key) { far_store(&st.cand[min(at, (uint32_t)kCand - 1u)], key); });
    if (!last_to_arrive(s, &st.arrived[1])) return;
    for (uint32_t i = threadIdx.x; i < n; i += kSampThreads) s.cand[i] = far_load(&st.cand[i]);
    __syncthreads();
    resolve_few(s, p, row, r, plan);
}

// One workgroup a row.
template <int DT>
__global__ void __launch_bounds__(kSampThreads) sample_rows_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t lds[];
    SampleLds &s = *reinterpret_cast<SampleLds *>(lds);
    const int row = blockIdx.x;
    const uint4 *base;
    int phase;
    const int pieces = row_pieces<DT>(p, row, base, phase);
    const float top = block_max(s, largest<DT>(p, base, phase, 0, pieces));
    if (top == -INFINITY) {                                // nothing can be chosen
        if (threadIdx.x == 0) no_token(p, row);
        return;
    }
    const RowRule r = row_rule(p, row, top);
    if (r.top_k == 1) {
        const uint32_t best = first_largest<DT>(s, p, base, phase, 0, pieces, top);
        if (threadIdx.x == 0) only_token(p, row, best);
        return;
    }
    if (threadIdx.x == 0) { s.top = top; s.n_cand = 0; }
    fill_base(s);
    histogram<DT>(s, p, r, base, phase, 0, pieces, top);
    const MyBins mine = scan_bins(s, [&](int i, uint64_t &m, uint32_t &c) { m = s.mass[i]; c = s.count[i]; });
    const RowPlan plan = make_plan(s, mine, r, top);
    if (plan.gathered > kCand) {
        resolve_many<DT>(s, p, row, r, plan);
        return;
    }
    gather<DT>(s, p, r, plan, base, phase, 0, pieces, [&](uint32_t n) { return take(&s.n_cand, n); },
               [&](uint32_t at, uint64_t key) { s.cand[min(at, (uint32_t)kCand - 1u)] = key; });
    __syncthreads();
    resolve_few(s, p, row, r, plan);
}

// Slices a row: as many as make one round of 256 workgroups (one a CU), of 4096 logits or more.  A workgroup for the whole row (one
// launch) where slices would take fewer than 44 k of the row's logits off it.  us, fp32, no filters, one workgroup / slices:
// 1 x 32003 19.6 / 18.9, 64 x 32003 19.9 / 25.5, 64 x 50257 26.0 / 27.5, 128 x 65537 36.4 / 40.8, 128 x 100003 51.6 / 53.9,
// 1 x 50257 23.9 / 18.4, 64 x 65537 31.0 / 29.2, 64 x 151936 69.6 / 45.8, 1 x 151936 56.5 / 19.2; 200 x 151936 83.4 / (two rounds) 111.
static int sample_slices(const pkv_sample_args *a) {
    int g = 256 / a->rows;
    g = g < a->vocab / 4096 ? g : a->vocab / 4096;
    g = g < kMaxSlices ? g : kMaxSlices;
    return g < 2 || a->vocab - a->vocab / g < 44 * 1024 ? 1 : g;
}

static int sample_check(const pkv_sample_args *a) {
    PKV_REQUIRE(a != nullptr, PKV_ERR_INVALID, "null pointer argument");
    PKV_REQUIRE(a->dtype == PKV_F16 || a->dtype == PKV_BF16 || a->dtype == PKV_F32, PKV_ERR_UNSUPPORTED, "Unsupported data type");
    PKV_REQUIRE(a->rows > 0 && a->vocab > 0, PKV_ERR_INVALID, "sizes must be positive");
    PKV_REQUIRE(a->rows < (1 << 22), PKV_ERR_UNSUPPORTED, "not supported: %d rows (fewer than 2^22)", a->rows);        // (2^32 threads)
    PKV_REQUIRE(a->vocab <= (1 << 20), PKV_ERR_UNSUPPORTED, "not supported: %d tokens (at most 2^20)", a->vocab);
    return PKV_OK;
}

template <class K> static hipError_t sample_lds(K kernel) {
    return hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SampleLds));
}
template <int DT> static int sample_launch(const SampleParams &p, int slices, void *workspace, hipStream_t s) {
    if (slices == 1) {
        PKV_HIP_CHECK(sample_lds(sample_rows_kernel<DT>));
        sample_rows_kernel<DT><<<dim3((unsigned)p.rows), kSampThreads, sizeof(SampleLds), s>>>(p);
    } else {
        RowState *state = (RowState *)workspace;
        const dim3 grid((unsigned)slices, (unsigned)p.rows);
        PKV_HIP_CHECK(sample_lds(slice_histogram_kernel<DT>));
        PKV_HIP_CHECK(sample_lds(slice_resolve_kernel<DT>));
        slice_top_kernel<DT><<<grid, kSampThreads, 0, s>>>(p, state);
        slice_histogram_kernel<DT><<<grid, kSampThreads, sizeof(SampleLds), s>>>(p, state);
        slice_resolve_kernel<DT><<<grid, kSampThreads, sizeof(SampleLds), s>>>(p, state);
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
