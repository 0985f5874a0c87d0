// snk_sample.hip — one index a row from logits: temperature, top-k, top-p, min-p and a given random
// number (include/snakehip.h states the rules).
//
// Every filter keeps a prefix of the order (x descending, equal ones by lower index), so a row's
// answer needs no sort: the prefix is a cut (key kt, nt): the entries above kt and the first nt of
// the entries equal to it, in index order. Masses inside a row's cut are integers (weights rounded to
// 2^-sh of the largest), so sums in LDS atomics are exact and always the same.
//
// Rows of up to 8 entries take a thread each (sample_few_kernel), of up to 4,096 the registers of one to
// four waves (sample_wave_kernel).
// A longer row is read once for what decides most rows: the largest logit of every 64 (a bound for top-k and
// min-p) and, where the whole row's mass counts, the mass of every 2048 (sample_scan_kernel). For
// top-p alone two more passes over the row find the cut's neighbourhood and the masses above it
// (sample_bins_kernel, sample_kept_kernel). The row's workgroup (sample_row_kernel) then reads only
// what can hold the answer. A few rows of up to 8,192 are scanned by that workgroup itself.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "snk_dqn.hpp"

namespace snk {

constexpr int PIECE = 512;      // consecutive elements a wave reads at once: 8 a lane
constexpr int GROUP = 64;       // elements of a recorded maximum: 8 lanes' worth
constexpr int GP = PIECE / GROUP;
constexpr int BP = 4;           // pieces of a block, the scan's unit of mass
constexpr int BLOCK = BP * PIECE;
constexpr int BINS = 2048;      // of a level of the radix search: 11 + 11 + 10 bits of the key
constexpr int NUCLEUS_LIST = 512;   // candidates that top-p alone lists where no other search was run
constexpr int NBINS = 1024;     // of the nucleus' mass over the distance from the top
constexpr int NLIST = 512;      // most entries of the cut's bin that one split of a row lists
constexpr int SPLITS = 16;      // most splits of a row

struct SampleHead {             // the nucleus search's results
    double sum;                 // by sample_bins_kernel: the row's mass in units, the largest entry,
    float top, step;            // bins a unit of distance
    int32_t fine, ok;           // a finite top and a mass to go by; a bin was found
    uint64_t above;             // by sample_kept_kernel: mass over the bin
};
struct SampleArgs {
    const void *x;
    int64_t rows, ld, ld_mask;
    int32_t n;
    const uint8_t *mask;
    const float *u;
    float temperature, top_p, min_p;
    int32_t top_k;
    const float *t_dev, *p_dev, *q_dev;
    const int32_t *k_dev;
    int32_t *idx;
    float *prob;
    double unit;              // 2^sh
    // the policy over an env batch: u from the counter RNG, the answer as an action
    uint8_t *act;
    uint64_t seed;
    const int64_t *tptr;
    // the scan's records (workspace), [rows][blocks]: masses relative to the block's largest entry,
    // that entry, and the maxima of 64
    double *masses;
    float *block_tops, *tops;
    int64_t row0;   // the first row of this launch
    // top-p alone: each row in `splits` parts
    int32_t splits;
    uint64_t *bins, *kept;    // [row][split][NBINS], [row][blocks]
    uint2 *lists;             // [row][split][NLIST] key, index
    uint32_t *listed;         // [row][split]
    SampleHead *heads;        // [row]; nullptr: not run
};

// a row's settings, the same for all its threads
struct SampleRow {
    double t, inv_t;
    bool greedy;
    int k;        // 1..n
    float p, q, u;
    // whether the mass of the whole row is needed
    __device__ __forceinline__ bool whole(int n) const { return k == n && (p < 1.0f || q == 0.0f); }
    __device__ __forceinline__ bool nucleus(int n) const { return k == n && p < 1.0f; }   // top-p alone
};
__device__ __forceinline__ SampleRow sample_row(const SampleArgs &A, int64_t r) {
    SampleRow s;
    const float t = A.t_dev ? A.t_dev[r] : A.temperature;
    s.greedy = !(t > 0.0f);
    s.t = s.greedy ? 1.0 : fmin((double)t, 1e300);   // t = inf: all alike, -inf still nothing
    s.inv_t = 1.0 / s.t;
    const int k = A.k_dev ? A.k_dev[r] : A.top_k;
    s.k = s.greedy ? 1 : k > 0 && k < A.n ? k : A.n;
    const float p = A.p_dev ? A.p_dev[r] : A.top_p, q = A.q_dev ? A.q_dev[r] : A.min_p;
    s.p = p < 1.0f && !s.greedy ? fmaxf(p, 0.0f) : 1.0f;   // NaN: off
    s.q = q > 0.0f ? fminf(q, 1.0f) : 0.0f;
    const float u = A.u ? A.u[r] : rng_uniform(rng_hash(A.seed, (uint64_t)r, (uint64_t)*A.tptr));
    s.u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    return s;
}

// order-preserving key of an allowed logit; 0 for -inf (excluded)
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 becomes +0: they are equal
    return x == -INFINITY ? 0u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The bits of 2^(j/128) less j 2^45: adding i 2^45, i = 128 e + j, gives those of 2^(e + j/128)
// without splitting i
__device__ const uint64_t POW2[128] = {
    0x3ff0000000000000ull, 0x3feff63da9fb3335ull, 0x3fefec9a3e778061ull, 0x3fefe315e86e7f85ull,
    0x3fefd9b0d3158574ull, 0x3fefd06b29ddf6deull, 0x3fefc74518759bc8ull, 0x3fefbe3ecac6f383ull,
    0x3fefb5586cf9890full, 0x3fefac922b7247f7ull, 0x3fefa3ec32d3d1a2ull, 0x3fef9b66affed31bull,
    0x3fef9301d0125b51ull, 0x3fef8abdc06c31ccull, 0x3fef829aaea92de0ull, 0x3fef7a98c8a58e51ull,
    0x3fef72b83c7d517bull, 0x3fef6af9388c8deaull, 0x3fef635beb6fcb75ull, 0x3fef5be084045cd4ull,
    0x3fef54873168b9aaull, 0x3fef4d5022fcd91dull, 0x3fef463b88628cd6ull, 0x3fef3f49917ddc96ull,
    0x3fef387a6e756238ull, 0x3fef31ce4fb2a63full, 0x3fef2b4565e27cddull, 0x3fef24dfe1f56381ull,
    0x3fef1e9df51fdee1ull, 0x3fef187fd0dad990ull, 0x3fef1285a6e4030bull, 0x3fef0cafa93e2f56ull,
    0x3fef06fe0a31b715ull, 0x3fef0170fc4cd831ull, 0x3feefc08b26416ffull, 0x3feef6c55f929ff1ull,
    0x3feef1a7373aa9cbull, 0x3feeecae6d05d866ull, 0x3feee7db34e59ff7ull, 0x3feee32dc313a8e5ull,
    0x3feedea64c123422ull, 0x3feeda4504ac801cull, 0x3feed60a21f72e2aull, 0x3feed1f5d950a897ull,
    0x3feece086061892dull, 0x3feeca41ed1d0057ull, 0x3feec6a2b5c13cd0ull, 0x3feec32af0d7d3deull,
    0x3feebfdad5362a27ull, 0x3feebcb299fddd0dull, 0x3feeb9b2769d2ca7ull, 0x3feeb6daa2cf6642ull,
    0x3feeb42b569d4f82ull, 0x3feeb1a4ca5d920full, 0x3feeaf4736b527daull, 0x3feead12d497c7fdull,
    0x3feeab07dd485429ull, 0x3feea9268a5946b7ull, 0x3feea76f15ad2148ull, 0x3feea5e1b976dc09ull,
    0x3feea47eb03a5585ull, 0x3feea34634ccc320ull, 0x3feea23882552225ull, 0x3feea155d44ca973ull,
    0x3feea09e667f3bcdull, 0x3feea012750bdabfull, 0x3fee9fb23c651a2full, 0x3fee9f7df9519484ull,
    0x3fee9f75e8ec5f74ull, 0x3fee9f9a48a58174ull, 0x3fee9feb564267c9ull, 0x3feea0694fde5d3full,
    0x3feea11473eb0187ull, 0x3feea1ed0130c132ull, 0x3feea2f336cf4e62ull, 0x3feea427543e1a12ull,
    0x3feea589994cce13ull, 0x3feea71a4623c7adull, 0x3feea8d99b4492edull, 0x3feeaac7d98a6699ull,
    0x3feeace5422aa0dbull, 0x3feeaf3216b5448cull, 0x3feeb1ae99157736ull, 0x3feeb45b0b91ffc6ull,
    0x3feeb737b0cdc5e5ull, 0x3feeba44cbc8520full, 0x3feebd829fde4e50ull, 0x3feec0f170ca07baull,
    0x3feec49182a3f090ull, 0x3feec86319e32323ull, 0x3feecc667b5de565ull, 0x3feed09bec4a2d33ull,
    0x3feed503b23e255dull, 0x3feed99e1330b358ull, 0x3feede6b5579fdbfull, 0x3feee36bbfd3f37aull,
    0x3feee89f995ad3adull, 0x3feeee07298db666ull, 0x3feef3a2b84f15fbull, 0x3feef9728de5593aull,
    0x3feeff76f2fb5e47ull, 0x3fef05b030a1064aull, 0x3fef0c1e904bc1d2ull, 0x3fef12c25bd71e09ull,
    0x3fef199bdd85529cull, 0x3fef20ab5fffd07aull, 0x3fef27f12e57d14bull, 0x3fef2f6d9406e7b5ull,
    0x3fef3720dcef9069ull, 0x3fef3f0b555dc3faull, 0x3fef472d4a07897cull, 0x3fef4f87080d89f2ull,
    0x3fef5818dcfba487ull, 0x3fef60e316c98398ull, 0x3fef69e603db3285ull, 0x3fef7321f301b460ull,
    0x3fef7c97337b9b5full, 0x3fef864614f5a129ull, 0x3fef902ee78b3ff6ull, 0x3fef9a51fbc74c83ull,
    0x3fefa4afa2a490daull, 0x3fefaf482d8e67f1ull, 0x3fefba1bee615a27ull, 0x3fefc52b376bba97ull,
    0x3fefd0765b6e4540ull, 0x3fefdbfdad9cbe14ull, 0x3fefe7c1819e90d8ull, 0x3feff3c22b8f71f1ull,
};

// e^((x - top) / T) by a table and a short polynomial (Tang 1989), to 3e-12: a u that falls between the sums of two evaluations that near is a one in
// 10^5 event over a row of 10^5 entries. 2^(i + j/128 + f/128), |f| <= 1/2: a table in LDS, a cubic,
// and the exponent added to the table's: 15 instructions, a quarter of the library's exp. Entries
// behind 2^-1000 (-inf too) weigh that much: callers leave excluded ones out themselves.
typedef const __attribute__((address_space(3))) uint64_t *LdsTable;   // no generic pointer's checks per look-up
struct Scale {
    double scale, low;   // 128 log2(e) / T, and the distance at which the weight is 2^-1000
};
__device__ __forceinline__ double exp_weight(double d, Scale S, LdsTable pow2) {   // 2^(d scale / 128), d <= 0
    d = fmax(d, S.low);
    const double t = fma(d, S.scale, 0x1.8p52), f = fma(d, S.scale, 0x1.8p52 - t);   // t's low word: d scale rounded
    const int i = __double2loint(t);
    // (ln 2 / 128)^k / k!
    double e = fma(f, 0x1.c6b08d704a0bfp-26, 0x1.ebfbdff82c58ep-17);
    e = fma(f, e, 0x1.62e42fefa39efp-8);
    const uint64_t p = pow2[i & 127];
    const double m = __hiloint2double((int)((uint32_t)(p >> 32) + ((uint32_t)i << 13)), (int)(uint32_t)p);
    return fma(m, f * e, m);
}
struct Weight {
    LdsTable pow2;        // copy of POW2
    double top;
    Scale scale;
    double unit;
    bool hard;   // only entries equal to the largest weigh: temperature 0, or +inf among them
    __device__ __forceinline__ double soft(float x) const { return exp_weight((double)x - top, scale, pow2); }
    __device__ __forceinline__ double real(float x) const {
        if (hard) return (double)x == top ? 1.0 : 0.0;
        return soft(x);
    }
    // w unit rounded to a whole number: w unit <= 2^51, so that adding 2^52 leaves it in the low bits
    __device__ __forceinline__ uint64_t fixed(double w) const {
        return (uint64_t)__double_as_longlong(fma(w, unit, 0x1p52)) & 0xFFFFFFFFFFFFFull;
    }
};
__device__ __forceinline__ Scale scale_of(const SampleRow &s) {
    return Scale{s.inv_t * 0x1.71547652b82fep+7, s.t * -693.0};
}
__device__ __forceinline__ Weight weight(const SampleArgs &A, const SampleRow &s, LdsTable pow2, float top) {
    return Weight{pow2, (double)top, scale_of(s), A.unit, s.greedy || top == INFINITY};
}

template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Packed {
    T v[V];
};
// Elements i..i+V-1 of a row of n >= V, -inf where masked or behind the end. In two steps, so that several loads are in flight before one is waited for: the load, of a
// whole vector inside the row whatever i is, and the values, by single elements where it was moved.
template <class T, int V = 8>
struct Raw {
    Packed<T, V> q;
    Packed<uint8_t, V> m;
    __device__ __forceinline__ void load(const T *x, const uint8_t *mask, int i, int n) {
        const int at = min(i, n - V);
        q = *reinterpret_cast<const Packed<T, V> *>(x + at);
        if (mask) m = *reinterpret_cast<const Packed<uint8_t, V> *>(mask + at);
    }
    __device__ __forceinline__ void values(const T *x, const uint8_t *mask, int i, int n, float *v) const {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = (float)q.v[k];
        if (mask) {
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = m.v[k] ? -INFINITY : v[k];
        }
        if (__any(i + V > n)) {   // a row's last vectors
            if (i + V > n)
#pragma unroll
                for (int k = 0; k < V; ++k)
                    v[k] = i + k < n && !(mask && mask[i + k]) ? (float)x[i + k] : -INFINITY;
        }
    }
};
template <class T>
__device__ __forceinline__ void load8(const T *x, const uint8_t *mask, int i, int n, float *v) {
    Raw<T> r;
    r.load(x, mask, i, n);
    r.values(x, mask, i, n, v);
}
template <int P, class T>
__device__ __forceinline__ void load_pieces(const T *x, const uint8_t *mask, int i, int n, float (*v)[8]) {
    Raw<T> r[P];
#pragma unroll
    for (int p = 0; p < P; ++p) r[p].load(x, mask, i + p * PIECE, n);
#pragma unroll
    for (int p = 0; p < P; ++p) r[p].values(x, mask, i + p * PIECE, n, v[p]);
}
// one element, likewise
template <class T>
struct Raw1 {
    T q;
    uint8_t m;
    __device__ __forceinline__ void load(const T *x, const uint8_t *mask, int i, int n) {
        const int at = min(i, n - 1);
        q = x[at];
        m = mask ? mask[at] : 0;
    }
    __device__ __forceinline__ float value(int i, int n) const { return i < n && !m ? (float)q : -INFINITY; }
};

// v + v of the lane that CTRL names in the lanes of rows ROWS, v alone in the others
template <class V, int CTRL, int ROWS>
__device__ __forceinline__ V dpp_add(V v) {
    constexpr int N = sizeof(V) / 4;
    union {
        V v;
        int w[N];
    } a, b;
    a.v = v;
#pragma unroll
    for (int i = 0; i < N; ++i) b.w[i] = __builtin_amdgcn_update_dpp(0, a.w[i], CTRL, ROWS, 0xf, false);
    return v + b.v;
}
// inclusive prefix over the wave, always in the same order: six steps of lane moves, no LDS
template <class V>
__device__ __forceinline__ V wave_scan(V v) {
    v = dpp_add<V, 0x111, 0xf>(v);   // row_shr 1, 2, 4, 8: within 16 lanes
    v = dpp_add<V, 0x112, 0xf>(v);
    v = dpp_add<V, 0x114, 0xf>(v);
    v = dpp_add<V, 0x118, 0xf>(v);
    v = dpp_add<V, 0x142, 0xa>(v);   // row_bcast 15: into rows 1 and 3
    return dpp_add<V, 0x143, 0xc>(v);   // row_bcast 31: into rows 2 and 3
}
template <class V>
__device__ __forceinline__ V read_lane(V v, int lane) {   // lane: the same on every lane
    constexpr int N = sizeof(V) / 4;
    union {
        V v;
        int w[N];
    } a;
    a.v = v;
#pragma unroll
    for (int i = 0; i < N; ++i) a.w[i] = __builtin_amdgcn_readlane(a.w[i], lane);
    return a.v;
}
template <class V>
__device__ __forceinline__ V last_lane(V v) {
    return read_lane(v, 63);
}
template <class V>
__device__ __forceinline__ V wave_sum(V v) {
    return last_lane(wave_scan(v));
}
template <int CTRL>
__device__ __forceinline__ float dpp_max(float x) {   // for lane moves that have a source for every lane
    return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true)));
}
__device__ __forceinline__ float max8(float x) {   // over each 8 lanes
    x = dpp_max<0xB1>(x);      // lanes ^ 1
    x = dpp_max<0x4E>(x);      // lanes ^ 2
    return dpp_max<0x141>(x);  // mirrored in 8
}
__device__ __forceinline__ float max64(float x) {   // of max8's
    x = dpp_max<0x140>(x);     // mirrored in 16
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}

__device__ __forceinline__ void answer(const SampleArgs &A, int64_t r, int i, double prob) {
    if (A.act) {
        A.act[r] = (uint8_t)(i < 0 ? 0 : i);
        return;
    }
    A.idx[r] = i;
    if (A.prob) A.prob[r] = (float)prob;
}

// records of the P pieces v that a wave holds: the maxima of 64 (NaN where one is among them), the
// largest entry and, with_mass, the sum of the weights relative to it
template <int P>
__device__ __forceinline__ void wave_records(const float (*v)[8], bool with_mass, Scale scale, LdsTable pow2,
                                             float *tops, float *top_out, double *mass) {
    const int lane = threadIdx.x & 63;
    float top = -INFINITY;
    uint64_t any_nan = 0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        float t = v[p][0];
        bool nan = t != t;
#pragma unroll
        for (int e = 1; e < 8; ++e) {
            nan |= v[p][e] != v[p][e];
            t = fmaxf(t, v[p][e]);
        }
        t = max8(nan ? -INFINITY : t);
        const uint64_t nans = __ballot(nan);
        any_nan |= nans;
        if ((lane & 7) == 0) tops[p * GP + (lane >> 3)] = (nans >> lane) & 255 ? NAN : t;
        top = fmaxf(top, t);
    }
    if (!with_mass && !top_out) return;
    top = max64(top);
    if (top_out && lane == 0) *top_out = any_nan ? NAN : top;
    if (!with_mass) return;
    double m = 0.0;
    if (top != -INFINITY && !any_nan) {
        if (top == INFINITY) {
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int e = 0; e < 8; ++e) m += v[p][e] == top ? 1.0 : 0.0;
        } else {
            const double wide = (double)top;   // subtracted, not folded into a fused product: exact for equal entries
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int e = 0; e < 8; ++e) m += exp_weight((double)v[p][e] - wide, scale, pow2);
        }
    }
    m = wave_sum(m);
    if (lane == 0) *mass = m;
}

// ---------------------------------------------------------------- the scan: a wave a block
// 2,048 entries a wave, four 16-byte loads a lane in flight before the first is waited for. With masses
// the weights bound it, 23 fp64 instructions an entry: 256 rows of 131,072 bf16 in 26 us, 2.6 TB/s,
// 22 us of them issue. Without (top-k, min-p alone) the reads: 512 rows of 32,003 bf16 8-10 us, 3.2 TB/s
// and more. The next block read ahead cost more in waves a SIMD than it hid.
template <class T>
__global__ __launch_bounds__(256) void sample_scan_kernel(SampleArgs A, int blocks, int64_t total) {
    __shared__ uint64_t pow2[128];
    if (threadIdx.x < 128) pow2[threadIdx.x] = POW2[threadIdx.x];
    __syncthreads();
    const int lane = threadIdx.x & 63;
    for (int64_t k = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); k < total;
         k += (int64_t)gridDim.x * 4) {
        const int64_t r = k / blocks;
        const int b = (int)(k - r * blocks);
        const SampleRow s = sample_row(A, r);
        const T *x = (const T *)A.x + r * A.ld;
        const uint8_t *mask = A.mask ? A.mask + r * A.ld_mask : nullptr;
        float v[BP][8];
        load_pieces<BP>(x, mask, b * BLOCK + lane * 8, A.n, v);
        wave_records<BP>(v, s.whole(A.n), scale_of(s), (LdsTable)pow2, A.tops + k * (BP * GP), A.block_tops + k, A.masses + k);
    }
}

// exclusive prefix of v over the threads of RW waves; total: of all. sh: RW + 1 values
template <int RW, class V>
__device__ __forceinline__ V block_scan(V v, V *sh, V &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const V in = wave_scan(v);
    __syncthreads();
    if (lane == 63) sh[wave] = in;
    __syncthreads();
    // every wave scans the waves' sums itself, within 16 lanes
    V sums = lane < RW ? sh[lane] : 0;
    sums = dpp_add<V, 0x111, 0xf>(sums);
    sums = dpp_add<V, 0x112, 0xf>(sums);
    if (RW > 4) {
        sums = dpp_add<V, 0x114, 0xf>(sums);
        sums = dpp_add<V, 0x118, 0xf>(sums);
    }
    total = read_lane(sums, RW - 1);
    const int w = __builtin_amdgcn_readfirstlane(wave);
    return (w ? read_lane(sums, w - 1) : V(0)) + (in - v);
}

template <int RW, class V>
__device__ __forceinline__ V block_sum(V v, V *sh) {
    V all;
    block_scan<RW, V>(v, sh, all);
    return all;
}

// ---------------------------------------------------------------- top-p alone
// The nucleus' cut is searched by mass over NBINS equal steps of the distance from the top, up to
// the distance at which an entry is sure to be outside: all entries lighter than e weigh less than
// n e together, so with n e = (1 - p) S none of them is in the nucleus.
struct Nucleus {
    float top, step;    // step: bins a unit of distance
    double sum;         // S in units
    bool ok;            // a finite top and a mass to go by
    __device__ __forceinline__ int bin(float x) const {   // NBINS: outside, or excluded
        const float b = (top - x) * step;
        return b < (float)NBINS ? (int)b : NBINS;
    }
};
// by the threads of one wave, from the scan's records of a row
__device__ __forceinline__ Nucleus nucleus(const SampleArgs &A, const SampleRow &s, LdsTable pow2, int64_t r, int blocks) {
    const int lane = threadIdx.x & 63;
    const float *bt = A.block_tops + r * blocks;
    float top = -INFINITY;
    bool nan = false;
    for (int b = lane; b < blocks; b += 64) {
        nan |= bt[b] != bt[b];
        top = fmaxf(top, bt[b]);
    }
    top = max64(max8(top));
    Nucleus N{};
    N.top = top;
    N.ok = !__ballot(nan) && fabsf(top) < INFINITY;
    if (!N.ok) return N;
    const Weight W = weight(A, s, (LdsTable)pow2, top);
    double sum = 0.0;
    for (int b = lane; b < blocks; b += 64)
        if (bt[b] != -INFINITY) sum += A.masses[r * blocks + b] * W.soft(bt[b]);
    sum = wave_sum(sum);
    N.sum = sum * A.unit;
    // the hardware's log2 (1 ulp), a little further out; its argument is at least 1: sum <= n
    const float far = __builtin_amdgcn_logf((float)A.n / ((float)(1.0 - (double)s.p) * (float)sum)) * 0.69315f + 1e-3f;
    N.step = NBINS / far * (float)s.inv_t;
    N.ok = N.step < INFINITY && N.step > 0.0f;
    return N;
}

// A workgroup a split of a row, a wave a piece: its mass by bins. Rows are split until the card has 1,024
// workgroups, a row into 16 at most (8 rows of 131,072 fp32: 6.9 us, the kernel after it 8.7). Bound by
// the LDS atomics of neighbours that meet in one bin and, with few rows, by one wave's chain of steps.
constexpr int NW = 16, NTH = 64 * NW;
static_assert(NBINS == NTH && NW % BP == 0, "a bin a thread, whole blocks a round");
template <class T>
__global__ __launch_bounds__(1024) void sample_bins_kernel(SampleArgs A, int blocks) {
    __shared__ uint64_t pow2[128];
    __shared__ uint64_t mass[NBINS];
    const int64_t r = A.row0 + blockIdx.x / A.splits;
    const int part = blockIdx.x % A.splits, tid = threadIdx.x, lane = tid & 63;
    const SampleRow s = sample_row(A, r);
    if (!s.nucleus(A.n)) return;
    const T *x = (const T *)A.x + r * A.ld;
    const uint8_t *mask = A.mask ? A.mask + r * A.ld_mask : nullptr;
    const int per = (blocks + A.splits - 1) / A.splits * BP, end = min((part + 1) * per, blocks * BP);   // pieces
    int c = part * per + __builtin_amdgcn_readfirstlane(tid >> 6);
    Raw<T> raw;   // of the next piece: in flight during all that follows
    if (c < end) raw.load(x, mask, c * PIECE + lane * 8, A.n);
    if (tid < 128) pow2[tid] = POW2[tid];
    mass[tid] = 0;
    __syncthreads();
    const Nucleus N = nucleus(A, s, (LdsTable)pow2, r, blocks);
    if (part == 0 && tid == 0) {
        SampleHead &head = A.heads[r - A.row0];
        head.sum = N.sum;
        head.top = N.top;
        head.step = N.step;
        head.fine = N.ok;
    }
    if (!N.ok) return;
    const Weight W = weight(A, s, (LdsTable)pow2, N.top);
    for (; c < end; c += NW) {
        float v[8];
        raw.values(x, mask, c * PIECE + lane * 8, A.n, v);
        if (c + NW < end) raw.load(x, mask, (c + NW) * PIECE + lane * 8, A.n);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int k = N.bin(v[e]);
            if (k < NBINS) atomicAdd((unsigned long long *)&mass[k], (unsigned long long)W.fixed(W.soft(v[e])));
        }
    }
    __syncthreads();
    A.bins[(int64_t)blockIdx.x * NBINS + tid] = mass[tid];
}

// the same split once more: the cut's bin, the masses of its blocks above that bin (and not under
// min-p), and the bin's entries
template <class T>
__global__ __launch_bounds__(1024) void sample_kept_kernel(SampleArgs A, int blocks) {
    __shared__ uint64_t pow2[128];
    __shared__ uint64_t scan[NW];
    __shared__ int cut_bin;
    __shared__ uint64_t cut_above;
    __shared__ uint32_t listed;
    const int64_t local = blockIdx.x / A.splits, r = A.row0 + local;
    const int part = blockIdx.x % A.splits, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const SampleRow s = sample_row(A, r);
    if (!s.nucleus(A.n)) return;
    const T *x = (const T *)A.x + r * A.ld;
    const uint8_t *mask = A.mask ? A.mask + r * A.ld_mask : nullptr;
    const int per = (blocks + A.splits - 1) / A.splits * BP, end = min((part + 1) * per, blocks * BP);
    Raw<T> raw;
    if (part * per + wave < end) raw.load(x, mask, (part * per + wave) * PIECE + lane * 8, A.n);
    uint64_t m = 0, all;   // the bin of this thread, from the top
    const uint64_t *bins = A.bins + local * A.splits * NBINS + tid;
    const SampleHead &head = A.heads[local];
    const Nucleus N{head.top, head.step, head.sum, head.fine != 0};
    if (A.splits == 1) {
        m = bins[0];
    } else {   // all loads in flight at once: 10,000 cycles one after another
        uint64_t part_mass[SPLITS];
#pragma unroll
        for (int k = 0; k < SPLITS; ++k) part_mass[k] = bins[min(k, A.splits - 1) * NBINS];
#pragma unroll
        for (int k = 0; k < SPLITS; ++k) m += k < A.splits ? part_mass[k] : 0;
    }
    if (tid < 128) pow2[tid] = POW2[tid];
    if (tid == 0) {
        cut_bin = -1;
        listed = 0;
    }
    __syncthreads();
    if (N.ok) {
        const double limit = (double)s.p * N.sum;
        const uint64_t above = block_scan<NW, uint64_t>(m, scan, all);
        if ((above == 0 || (double)above < limit) && (double)(above + m) >= limit && m) {   // one bin
            cut_bin = tid;
            cut_above = above;
        }
    }
    __syncthreads();
    const int cut = cut_bin;
    if (part == 0 && tid == 0) {   // what no other workgroup reads yet
        A.heads[local].above = cut < 0 ? 0 : cut_above;
        A.heads[local].ok = cut >= 0;
    }
    if (cut < 0) return;
    const Weight W = weight(A, s, (LdsTable)pow2, N.top);
    const double q = (double)s.q;
    uint2 *list = A.lists + (int64_t)blockIdx.x * NLIST;
    for (int c0 = part * per; c0 < end; c0 += NW) {
        const int c = c0 + wave, i = c * PIECE + lane * 8;
        uint64_t sum = 0;
        if (c < end) {
            float v[8];
            raw.values(x, mask, i, A.n, v);
            if (c + NW < end) raw.load(x, mask, i + NW * PIECE, A.n);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = N.bin(v[e]);
                if (k < cut) {
                    const double w = W.soft(v[e]);
                    sum += w >= q ? W.fixed(w) : 0;
                } else if (k == cut) {
                    const uint32_t at = atomicAdd(&listed, 1u);
                    if (at < NLIST) list[at] = make_uint2(key_of(v[e]), (uint32_t)(i + e));
                }
            }
        }
        sum = wave_sum(sum);
        __syncthreads();
        if (lane == 0) scan[wave] = sum;
        __syncthreads();
        if (tid < NW / BP && c0 + tid * BP < end) {
            uint64_t block = 0;
#pragma unroll
            for (int p = 0; p < BP; ++p) block += scan[tid * BP + p];
            A.kept[local * blocks + c0 / BP + tid] = block;
        }
    }
    __syncthreads();
    if (tid == 0) A.listed[blockIdx.x] = listed;
}

// ---------------------------------------------------------------- a thread a row: n <= N
// Everything in registers, ranks by all pairs. 65,536 rows of 3 fp32: 4.0 us, 0.3 TB/s: a launch's own
// 3.6 us; a wave a row (the next kernel) 23 us.
template <class T, int N>
__global__ __launch_bounds__(256) void sample_few_kernel(SampleArgs A) {
    __shared__ uint64_t pow2[128];
    if (threadIdx.x < 128) pow2[threadIdx.x] = POW2[threadIdx.x];
    __syncthreads();
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= A.rows) return;
    const SampleRow s = sample_row(A, r);
    const T *x = (const T *)A.x + r * A.ld;
    const uint8_t *mask = A.mask ? A.mask + r * A.ld_mask : nullptr;
    float v[N], top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = i < A.n && !(mask && mask[i]) ? (float)x[i] : -INFINITY;
        nan |= v[i] != v[i];
        top = fmaxf(top, v[i]);
    }
    if (nan || top == -INFINITY) {
        answer(A, r, -1, nan ? NAN : 0.0);
        return;
    }
    const Weight W = weight(A, s, (LdsTable)pow2, top);
    uint64_t w[N], s1 = 0, sum = 0;
    int rank[N];
    bool kept[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const double wr = v[i] == -INFINITY ? 0.0 : W.real(v[i]);
        rank[i] = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) rank[i] += v[j] > v[i] || (v[j] == v[i] && j < i);
        kept[i] = v[i] != -INFINITY && rank[i] < s.k;
        w[i] = kept[i] ? W.fixed(wr) : 0;
        kept[i] = kept[i] && wr >= (double)s.q;
        s1 += w[i];
    }
    const double limit = (double)s.p * (double)s1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        uint64_t before = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) before += rank[j] < rank[i] ? w[j] : 0;
        kept[i] = kept[i] && (s.p >= 1.0f || rank[i] == 0 || (double)before < limit);
        sum += kept[i] ? w[i] : 0;
    }
    const double target = (double)s.u * (double)sum;
    uint64_t upto = 0;
    int at = -1;
    float xa = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        upto += kept[i] ? w[i] : 0;
        if (at < 0 && kept[i] && (double)upto > target) {
            at = i;
            xa = v[i];
        }
    }
    answer(A, r, at, W.real(xa) * A.unit / (double)sum);
}

// ---------------------------------------------------------------- 64 E NW threads' registers a row
// Comparisons with others that cost what one bit of a search by mass does. 65,536 rows, top-p 0.9, fp32
// (28 bits): n = 16 54 us by pairs and 190 by bits, n = 64 130 and 190; bf16 (13 bits): n = 48 104 and
// 111, n = 64 130 and 111.
constexpr int PAIRS_A_BIT = 4;
// Every so many bits of an fp32 search by mass, those that the keys still in question share are set at
// once: 32,768 rows, top-p 0.9, n = 128 69 us against 115, n = 1,024 214 against 253. 16-bit keys have too
// few bits for that (bf16, n = 1,024: 181 and 168).
constexpr int NARROW = 4;
// low bits that the keys of the type's positive values share, and those of its negative ones
template <class T>
constexpr int KEY_SHIFT = sizeof(T) == 4 ? 0 : std::is_same<T, __bf16>::value ? 16 : 13;

// Thread l of the row's holds the elements E l..E l + E - 1, so that a prefix over the row is E additions
// and one over the lanes. The cut's key is built from its highest bit that the row's keys differ in: by
// how many entries are not below it (top-k: E comparisons and bit counts), or by their mass (top-p).
// NW waves a row: alone (four rows a workgroup), or a workgroup, whose waves add up through LDS.
// Bound by its instructions, 20 an element for the weight and the prefix and 2 (top-k) or 5 (top-p) an
// element a bit. 65,536 rows of 1,024 bf16: 133 us whole, 225 top-k 40, 315 top-p 0.9 (a workgroup
// with bins and lists in LDS a row: 366, 1,097, 1,622); 256 rows: 10 us, of which 6 are the launch.
template <class T, int E, int NW>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void sample_wave_kernel(SampleArgs A) {
    constexpr int V = E < 8 ? E : 8, SHIFT = KEY_SHIFT<T>, ROWS = NW == 1 ? 4 : 1;
    __shared__ uint64_t pow2[128];
    __shared__ uint64_t slots[2][NW];   // one sum's while the last one's are read
    __shared__ float tops[NW];
    __shared__ uint32_t leasts[NW];
    __shared__ uint32_t list_key[ROWS][64], list_at[ROWS][64];
    if (threadIdx.x < 128) pow2[threadIdx.x] = POW2[threadIdx.x];
    __syncthreads();
    const int lane = threadIdx.x & 63, n = A.n, in_group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = NW == 1 ? 0 : in_group, i0 = (wave * 64 + lane) * E;
    const int64_t r = A.row0 + (int64_t)blockIdx.x * ROWS + (NW == 1 ? in_group : 0);
    if (r >= A.rows) return;
    const T *x = (const T *)A.x + r * A.ld;
    const uint8_t *mask = A.mask ? A.mask + r * A.ld_mask : nullptr;
    Raw<T, V> raw[E / V];
#pragma unroll
    for (int p = 0; p < E / V; ++p) raw[p].load(x, mask, i0 + p * V, n);
    const SampleRow s = sample_row(A, r);
    float v[E];
#pragma unroll
    for (int p = 0; p < E / V; ++p) raw[p].values(x, mask, i0 + p * V, n, v + p * V);
    uint32_t key[E];   // above SHIFT; 0: excluded
    float most = -INFINITY;
    uint32_t least = 0xFFFFFFFFu;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        nan |= v[e] != v[e];
        most = fmaxf(most, v[e]);
        key[e] = key_of(v[e]) >> SHIFT;
        least = min(least, key[e] - 1);   // 0 becomes the largest
    }
    float top = max64(max8(most));
    nan = __ballot(nan) != 0;
    const bool cut = s.k < n || s.p < 1.0f;
    if (cut)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) least = min(least, (uint32_t)__shfl_xor((int)least, o));
    if constexpr (NW > 1) {
        if (lane == 0) {
            tops[wave] = nan ? NAN : top;
            leasts[wave] = least;
        }
        __syncthreads();
#pragma unroll
        for (int o = 0; o < NW; ++o) {
            const float t = tops[o];
            nan |= t != t;
            top = fmaxf(top, t);
            least = min(least, leasts[o]);
        }
    }
    if (nan || top == -INFINITY) {   // all of the row's waves
        if (threadIdx.x % (64 * NW) == 0) answer(A, r, -1, nan ? NAN : 0.0);
        return;
    }
    const Weight W = weight(A, s, (LdsTable)pow2, top);
    auto logit = [&](uint32_t k) __attribute__((always_inline)) {
        return of_key(k << SHIFT | (SHIFT && !(k >> (31 - SHIFT)) ? (1u << SHIFT) - 1 : 0u));
    };
    uint64_t w[E];
    uint32_t heavy = 0;   // what min-p keeps, a bit an element
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const double real = key[e] ? W.real(v[e]) : 0.0;
        w[e] = W.fixed(real);
        heavy |= real >= (double)s.q ? 1u << e : 0u;
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // four at once: more only hold registers
    }
    int turn = 0;
    auto over_waves = [&](uint64_t mine, uint64_t &before) __attribute__((always_inline)) {   // mine: the wave's
        before = 0;
        if constexpr (NW == 1) return mine;
        if (lane == 0) slots[turn][wave] = mine;
        __syncthreads();
        uint64_t all = 0;
#pragma unroll
        for (int o = 0; o < NW; ++o) {
            const uint64_t m = slots[turn][o];
            before += o < wave ? m : 0;
            all += m;
        }
        turn ^= 1;
        return read_lane(all, 0);
    };
    auto not_below = [&](uint32_t at) __attribute__((always_inline)) {
        int c = 0;
        uint64_t before;
#pragma unroll
        for (int e = 0; e < E; ++e) c += __popcll(__ballot(key[e] >= at));
        return (int)over_waves((uint64_t)c, before);
    };
    auto mass_not_below = [&](uint32_t at) __attribute__((always_inline)) {
        uint64_t m = 0, before;
#pragma unroll
        for (int e = 0; e < E; ++e) m += key[e] >= at ? w[e] : 0;
        return over_waves(wave_sum(m), before);
    };
    // the row's largest and smallest of two values a lane
    auto span_over_waves = [&](uint32_t &most, uint32_t &least) __attribute__((always_inline)) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            most = max(most, (uint32_t)__shfl_xor((int)most, o));
            least = min(least, (uint32_t)__shfl_xor((int)least, o));
        }
        if constexpr (NW > 1) {
            if (lane == 0) slots[turn][wave] = (uint64_t)most << 32 | least;
            __syncthreads();
#pragma unroll
            for (int o = 0; o < NW; ++o) {
                const uint64_t m = slots[turn][o];
                most = max(most, (uint32_t)(m >> 32));
                least = min(least, (uint32_t)m);
            }
            turn ^= 1;
        }
        most = (uint32_t)__builtin_amdgcn_readfirstlane((int)most);
        least = (uint32_t)__builtin_amdgcn_readfirstlane((int)least);
    };
    auto key_weight = [&](uint32_t k) __attribute__((always_inline)) { return W.fixed(W.real(logit(k))); };
    // the first k of a wave's entries, one a lane in index order (key 0: none), their top-p and the
    // answer: each entry's rank and the mass before it by comparing it with the m others
    auto by_pairs = [&](uint32_t own_key, uint64_t own_w, bool over, int at, int m) __attribute__((always_inline)) {
        uint32_t ahead = 0;
        uint64_t mass = 0;
        for (int i = 0; i < m; ++i) {
            const uint32_t ki = read_lane(own_key, i);
            const bool before = (ki > own_key) | ((ki == own_key) & (i < lane));
            const uint64_t wi = read_lane(own_w, i);
            ahead += before;
            mass += before ? wi : 0;
        }
        bool kept = own_key && ahead < (uint32_t)s.k;
        const double limit = (double)s.p * (double)wave_sum<uint64_t>(kept ? own_w : 0);
        kept = kept && (s.p >= 1.0f || ahead == 0 || (double)mass < limit);
        const uint64_t w = kept && over ? own_w : 0, upto = wave_scan(w), sum = last_lane(upto);
        const double target = (double)s.u * (double)sum;
        if (w && (double)upto > target && !((double)(upto - w) > target))   // one lane
            answer(A, r, at, W.real(logit(own_key)) * A.unit / (double)sum);
    };
    // the cut: keys above kt, and the first nt of those equal to it
    uint32_t kt = 0, nt = 0;
    if (cut) {
        const uint32_t first = key_of(top) >> SHIFT;
        const uint32_t differ = (uint32_t)__builtin_amdgcn_readfirstlane((int)(first ^ (least + 1)));
        const int bits = differ ? 32 - __clz((int)differ) : 0;
        const uint32_t common = bits == 32 ? 0u : first >> bits << bits;
        if constexpr (E == 1 && NW == 1)
            if (s.p < 1.0f && n < PAIRS_A_BIT * bits) {
                by_pairs(key[0], w[0], heavy & 1, i0, n);
                return;
            }
        bool k_cut = false;
        if (s.k < n && not_below(1) > s.k) {
            k_cut = true;
            kt = common;
            int above = 0;
            for (int b = bits - 1; b >= 0; --b) {
                const uint32_t at = kt | 1u << b;
                const int c = not_below(at);
                if (c == s.k) {   // no tie is split
                    kt = at - 1;
                    above = c;
                    break;
                }
                if (c > s.k)
                    kt = at;
                else
                    above = c;   // at last: the entries over the key that the lower bits fill up to
            }
            nt = (uint32_t)(s.k - above);
        }
        if (E * NW > 1 && k_cut && s.k <= 64 && s.p < 1.0f) {
            // top-p over a wave's worth of entries: listed in index order, for one wave
            uint32_t ties = 0, mine = 0;
            uint64_t before;
#pragma unroll
            for (int e = 0; e < E; ++e) ties += key[e] == kt;
            uint32_t upto = wave_scan(ties);
            if constexpr (NW > 1) {
                over_waves(last_lane(upto), before);
                upto += (uint32_t)before;
            }
            uint32_t rank = upto - ties, in = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool is = key[e] > kt || (key[e] == kt && rank < nt);
                rank += key[e] == kt;
                in |= is ? 1u << e : 0u;
            }
            mine = (uint32_t)__popc(in);
            upto = wave_scan(mine);
            if constexpr (NW > 1) {
                over_waves(last_lane(upto), before);
                upto += (uint32_t)before;
            }
            uint32_t to = upto - mine;
            const int row = NW == 1 ? in_group : 0;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (in >> e & 1) {   // k in all
                    list_key[row][to] = key[e];
                    list_at[row][to++] = (uint32_t)(i0 + e);
                }
            if constexpr (NW > 1) {
                __syncthreads();
                if (wave != 0) return;
            } else {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the wave's own writes, then its reads
            }
            const uint32_t k = lane < s.k ? list_key[row][lane] : 0;
            const double real = k ? W.real(logit(k)) : 0.0;
            by_pairs(k, W.fixed(real), real >= (double)s.q, lane < s.k ? (int)list_at[row][lane] : -1, s.k);
            return;
        }
        if (s.p < 1.0f) {
            const uint64_t s1 = mass_not_below(kt + 1) + (nt ? nt * key_weight(kt) : 0);
            const double limit = (double)s.p * (double)s1;
            if (limit <= 0.0) {
                kt = first;
                nt = 1;
            } else {
                uint32_t t = common, over = first + 1;   // the cut's key is one of t..over - 1
                uint64_t above = 0;                      // mass from `over` on
                int steps = 0;
                for (int b = bits - 1; b >= 0; --b) {
                    const uint32_t at = t | 1u << b;
                    if (k_cut && at <= kt) {
                        t = at;
                        continue;
                    }
                    const uint64_t m = mass_not_below(at);
                    if ((double)m >= limit) {
                        t = at;
                    } else {
                        above = m;
                        over = at;
                    }
                    if (SHIFT == 0 && ++steps % NARROW == 0) {
                        uint32_t most = 0, least = 0xFFFFFFFFu;
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const bool in = key[e] >= t && key[e] < over;
                            most = max(most, in ? key[e] : 0u);
                            least = min(least, in ? key[e] : 0xFFFFFFFFu);
                        }
                        span_over_waves(most, least);
                        const uint32_t differ = most ^ least;
                        b = differ ? 32 - __clz((int)differ) : 0;
                        t = most >> b << b;   // a key is in question always, and four bits are known: b <= 28
                    }
                }
                // tie j stays while above + j w < limit
                const uint64_t wt = key_weight(t);
                const double more = wt ? ceil((limit - (double)above) / (double)wt) : (double)n;
                const uint32_t stay = (uint32_t)fmin(fmax(more, 1.0), (double)n);
                nt = k_cut && t == kt ? min(stay, nt) : stay;
                kt = t;
            }
        }
    }
    uint32_t rank = 0;
    if (nt) {
        uint32_t ties = 0;
        uint64_t before;
#pragma unroll
        for (int e = 0; e < E; ++e) ties += key[e] == kt;
        const uint32_t upto = wave_scan(ties);
        over_waves(last_lane(upto), before);
        rank = (uint32_t)before + upto - ties;
    }
    uint64_t own = 0, before;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        bool kept = key[e] > kt;
        if (nt && key[e] == kt) kept = rank++ < nt;
        w[e] = kept && (heavy >> e & 1) ? w[e] : 0;
        own += w[e];
    }
    uint64_t upto = wave_scan(own);
    const uint64_t sum = over_waves(last_lane(upto), before);
    upto += before;
    const double target = (double)s.u * (double)sum;
    if (own && (double)upto > target && !((double)(upto - own) > target)) {   // one lane of the row's
        upto -= own;
        int at = -1;
        uint32_t ka = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            upto += w[e];
            if (at < 0 && w[e] && (double)upto > target) {
                at = i0 + e;
                ka = key[e];
            }
        }
        answer(A, r, at, W.real(logit(ka)) * A.unit / (double)sum);
    }
}

// ---------------------------------------------------------------- a workgroup a row
// distance from the top by 64 steps an octave, 2^-12 .. 2^20: a bound that outliers do not spoil
__device__ __forceinline__ int far_bin(float d) {
    const int b = (int)(__float_as_uint(d) >> 17) - ((127 - 12) << 6);
    return min(max(b, 0), BINS - 1);
}
__device__ __forceinline__ float far_edge(int b) {   // all in bins up to b are nearer, and nothing else is
    return b < BINS - 1 ? __uint_as_float((uint32_t)(b + 1 + ((127 - 12) << 6)) << 17) : INFINITY;
}

// Bound by its chain of a dozen dependent steps between barriers, not by what it reads: 256 rows of
// 131,072 bf16, whole, 7.8 us; 128 of 50,021, top-k 40, 9.6; 8 of 131,072 fp32 after the nucleus search
// 12; 512 of 32,003, min-p 0.05, with 8 waves each 14 (4 us more with 16).
// OWN: pieces a wave scans here, 0: sample_scan_kernel's records
template <class T, int RW, int OWN>
__global__ __launch_bounds__(64 * RW) void sample_row_kernel(SampleArgs A) {
    constexpr bool FUSED = OWN > 0;
    constexpr int NT = 64 * RW, BT = BINS / NT;   // threads; bins of each
    constexpr int REC = FUSED ? OWN : BP;         // pieces of a record of mass
    // most candidates held in LDS, as many as leave room for the workgroups that the registers allow
    constexpr int LIST = RW == 16 ? 4096 : RW == 8 ? 2048 : 1024;
    static_assert(LIST * 4 <= BINS * 8, "group_list lies in mass");
    __shared__ uint64_t pow2[128];
    __shared__ uint64_t mass[BINS];
    __shared__ uint32_t count[BINS];
    __shared__ uint32_t list_key[LIST], list_at[LIST];
    __shared__ uint64_t scan64[RW];
    __shared__ double scanf[RW];
    __shared__ uint32_t scan32[RW];
    __shared__ float own_tops[FUSED ? RW * GP * OWN : 1];
    __shared__ double own_masses[FUSED ? RW : 1];
    __shared__ float wave_top[RW];
    __shared__ int wave_nan[RW];
    __shared__ uint64_t found_mass;
    __shared__ double found_sum;
    __shared__ uint32_t found_bin, found_count, listed;
    __shared__ double final_sum[4];
    __shared__ uint64_t final_mass[4];
    __shared__ uint32_t final_ties[4];
    __shared__ float final_x[4];
    __shared__ int final_last[4], final_hit[4];
    uint64_t *const seg_mass = mass;       // [NT], once the search is over
    uint32_t *const seg_ties = count;
    uint32_t *const group_list = (uint32_t *)mass;   // [LIST], before it
    const int64_t r = A.row0 + blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = A.n;
    const SampleRow s = sample_row(A, r);
    const T *x = (const T *)A.x + r * A.ld;
    const uint8_t *mask = A.mask ? A.mask + r * A.ld_mask : nullptr;
    const int pieces = (n + PIECE - 1) / PIECE, records = (pieces + REC - 1) / REC, groups = records * REC * GP;
    if (tid < 128) pow2[tid] = POW2[tid];
    if (tid == 0) listed = 0;
    const int per = (records + NT - 1) / NT, segs = (records + per - 1) / per;   // records a segment, segments

    // the nucleus search's results: loaded before what takes longer
    const int64_t local = blockIdx.x;
    SampleHead head{};
    uint32_t in_split = 0;
    uint64_t kept_above = 0;
    if (!FUSED && A.heads && s.nucleus(n)) {
        head = A.heads[local];
        in_split = lane < A.splits ? A.listed[local * A.splits + lane] : 0;
        if (tid < segs)
            for (int c = tid * per; c < min((tid + 1) * per, records); ++c) kept_above += A.kept[local * records + c];
    }

    const float *tops;
    const double *masses;
    if constexpr (FUSED) {
        __syncthreads();
        if (wave < records) {
            float v[OWN][8];
            load_pieces<OWN>(x, mask, wave * OWN * PIECE + lane * 8, n, v);
            wave_records<OWN>(v, s.whole(n), scale_of(s), (LdsTable)pow2, own_tops + wave * OWN * GP, nullptr, own_masses + wave);
        }
        __syncthreads();
        tops = own_tops;
        masses = own_masses;
    } else {
        tops = A.tops + r * groups;
        masses = A.masses + r * records;
    }
    const int share = (groups + NT - 1) / NT, g0 = tid * share, g1 = min(g0 + share, groups);   // consecutive groups a thread
    const float t_first = g0 < groups ? tops[g0] : -INFINITY;
    auto top_of = [&](int g) __attribute__((always_inline)) { return g == g0 ? t_first : tops[g]; };
    float top = -INFINITY;
    bool nan = false;
    const float *const top_src = FUSED ? tops : A.block_tops + r * records;
    for (int g = tid; g < (FUSED ? groups : records); g += NT) {
        const float t = top_src[g];
        nan |= t != t;
        top = fmaxf(top, t);
    }
    top = max64(max8(top));
    nan = __ballot(nan) != 0;
    if (lane == 0) {
        wave_top[wave] = top;
        wave_nan[wave] = nan;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        top = fmaxf(top, wave_top[w]);
        nan |= wave_nan[w] != 0;
    }
    if (nan || top == -INFINITY) {   // the whole workgroup
        if (tid == 0) answer(A, r, -1, nan ? NAN : 0.0);
        return;
    }
    const Weight W = weight(A, s, (LdsTable)pow2, top);
    const double q = (double)s.q;

    // the whole row's mass by segment, from the records
    double seg_sum = 0.0, sum_ex = 0.0, row_sum = 0.0;
    if (s.whole(n) && !head.ok) {
        if (tid < segs)
            for (int c = tid * per; c < min((tid + 1) * per, records); ++c) {
                float t;
                if constexpr (FUSED) {
                    t = tops[c * OWN * GP];
#pragma unroll
                    for (int g = 1; g < OWN * GP; ++g) t = fmaxf(t, tops[c * OWN * GP + g]);
                } else {
                    t = A.block_tops[r * records + c];
                }
                if (t != -INFINITY) seg_sum += masses[c] * W.real(t);
            }
        sum_ex = block_scan<RW, double>(seg_sum, scanf, row_sum);
    }

    // the cut: keys above kt, and the first nt of those equal to it
    uint32_t kt = 0, nt = 0;
    double target = 0.0, scale_out = 0.0;   // u S; the probability's 1 / S
    int seg = 0;
    uint64_t base = 0;
    uint32_t ties = 0;
    const bool cut = s.k < n || s.p < 1.0f, plain = !cut && q == 0.0;
    double base_real = 0.0;
    if (plain) {
        // nothing is filtered: the segment by the records' masses
        target = (double)s.u * row_sum;
        scale_out = 1.0 / row_sum;
        if (tid == 0) found_bin = 0;
        __syncthreads();
        // the last segment whose prefix is not over the target, of those that weigh anything
        if (seg_sum > 0.0 && !(sum_ex > target)) atomicMax(&found_bin, (uint32_t)tid);
        __syncthreads();
        if (tid == (int)found_bin) found_sum = sum_ex;
        __syncthreads();
        seg = (int)found_bin;
        base_real = found_sum;
    } else {
        const double limit_row = (double)s.p * (head.ok ? head.sum : row_sum * A.unit);   // top-p alone, in units
        bool use_list = true, binned = false;   // binned: the list is the cut's bin, the rest is above it
        uint64_t above_list = 0;
        if (!FUSED && A.heads && s.nucleus(n) && !W.hard) {
            bool fits = head.ok != 0;
            if (fits) {   // SPLITS <= 64: a lane a split, every wave for itself
                const uint32_t c = in_split;
                const uint32_t in = wave_scan(c), m = last_lane(in);
                fits = !__ballot(c > NLIST) && m <= LIST;
                for (int k = wave; k < A.splits && fits; k += RW) {
                    const uint32_t ck = (uint32_t)__builtin_amdgcn_readlane((int)c, k);
                    const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)in, k) - ck;
                    for (uint32_t i = lane; i < ck; i += 64) {
                        const uint2 e = A.lists[(local * A.splits + k) * NLIST + i];
                        list_key[at + i] = e.x;
                        list_at[at + i] = e.y;
                    }
                }
                if (tid == 0) listed = m;
            }
            binned = fits;
            use_list = fits;
            above_list = head.above;
        } else {
            // candidates: what can be in the cut, by the groups' maxima: bins of the distance from the
            // top up to here, and, where min-p is not to change the mass that top-p goes by, this near
            const bool by_q = s.q > 0.0f && s.p >= 1.0f;
            // (never 0, however low the temperature: the top itself is nearer)
            const float near = by_q ? fmaxf((__builtin_amdgcn_logf(s.q) * -0.69315f + 1e-4f) * (float)s.t, 0x1p-120f) : INFINITY;
            // Candidates are nearer to the top; NaN for two infinities: top itself. Without an edge all that is
            // allowed: a distance may be infinite in fp32 and yet weigh, where the temperature is as large, so
            // 0 stands for the top then.
            float edge, from;
            auto set_edge = [&](float e) __attribute__((always_inline)) {
                edge = e;
                from = e < INFINITY ? top : 0.0f;
            };
            set_edge(near);
            auto candidate = [&](float v) __attribute__((always_inline)) { return !(from - v >= edge); };
            bool dense = false;   // candidates in most groups
            if (W.hard) {
                set_edge(far_edge(0));
            } else if (cut) {
                // the bin that the wanted-th largest of the counted maxima falls in: at least that many
                // entries are as near
                uint32_t all, wanted;
                auto clear_counts = [&]() __attribute__((always_inline)) {
#pragma unroll
                    for (int b = 0; b < BT; ++b) count[b * NT + tid] = 0;
                    __syncthreads();
                };
                auto edge_by_counts = [&]() __attribute__((always_inline)) {
                    if (tid == 0) found_bin = BINS - 1;
                    __syncthreads();
                    uint32_t c[BT], sum = 0;
#pragma unroll
                    for (int b = 0; b < BT; ++b) sum += c[b] = count[tid * BT + b];
                    uint32_t ex = block_scan<RW, uint32_t>(sum, scan32, all);
                    // top-p alone: a list that most distributions' nucleus fits into
                    wanted = s.k < n ? (uint32_t)s.k : max(1u, min((uint32_t)NUCLEUS_LIST, all / 2));
#pragma unroll
                    for (int b = 0; b < BT; ++b) {
                        if (ex < wanted && ex + c[b] >= wanted) found_bin = tid * BT + b;
                        ex += c[b];
                    }
                    __syncthreads();
                    return fminf(near, far_edge((int)found_bin));
                };
                clear_counts();
                for (int g = g0; g < g1; ++g) {
                    const float t = top_of(g);
                    if (t != -INFINITY) atomicAdd(&count[far_bin(top - t)], 1u);
                }
                set_edge(edge_by_counts());
                // Too few groups for that many entries, or so few that their maxima leave more than the
                // list holds: of A groups, W with a larger maximum, -A ln(1 - W/A) entries are expected.
                // Then by the maxima of 8, read again: one row of 131,072, top-k 2,000, 39 us against 115 by a
                // radix search over the row, of 50,000, top-k 700 and top-p 0.9, 41 against 109.
                if (s.k < n && n > LIST && wanted <= LIST &&
                    (all <= wanted || (float)all * __logf(1.0f - (float)wanted / (float)all) < -0.85f * LIST)) {
                    dense = true;
                    clear_counts();
                    for (int c = wave * BP; c < pieces; c += RW * BP) {
                        float v[BP][8];
                        load_pieces<BP>(x, mask, c * PIECE + lane * 8, n, v);
#pragma unroll
                        for (int p = 0; p < BP; ++p) {
                            float t = v[p][0];
#pragma unroll
                            for (int e = 1; e < 8; ++e) t = fmaxf(t, v[p][e]);
                            if (t != -INFINITY) atomicAdd(&count[far_bin(top - t)], 1u);
                        }
                    }
                    set_edge(edge_by_counts());
                }
                // fewer maxima than wanted entries: everything would be a candidate
                use_list = all >= wanted || n <= LIST || by_q;
            }
            if (use_list && dense) {
                // a run of pieces a wave: its candidates counted, then listed
                const int run = (pieces + RW - 1) / RW, c0 = wave * run, c1 = min(c0 + run, pieces);
                auto each_piece = [&](auto &&f) __attribute__((always_inline)) {   // f(8 entries, the first's index)
                    for (int c = c0; c < c1; c += BP) {
                        float v[BP][8];
                        load_pieces<BP>(x, mask, c * PIECE + lane * 8, n, v);
#pragma unroll
                        for (int p = 0; p < BP; ++p)
                            if (c + p < c1) f(v[p], (c + p) * PIECE + lane * 8);
                    }
                };
                uint32_t own = 0;
                each_piece([&](const float *v, int) __attribute__((always_inline)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) own += candidate(v[e]);
                });
                own = wave_sum(own);
                if (lane == 0) scan32[wave] = own;
                __syncthreads();
                const uint32_t owns = wave_scan(lane < RW ? scan32[lane] : 0u);
                uint32_t at = wave ? read_lane(owns, wave - 1) : 0;
                if (tid == 0) listed = read_lane(owns, RW - 1);
                each_piece([&](const float *v, int i) __attribute__((always_inline)) {
                    uint32_t in = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) in += candidate(v[e]);
                    const uint32_t upto = wave_scan(in);
                    uint32_t to = at + upto - in;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (candidate(v[e])) {
                            if (to < LIST) {
                                list_key[to] = key_of(v[e]);
                                list_at[to] = (uint32_t)(i + e);
                            }
                            ++to;
                        }
                    at += last_lane(upto);
                });
            } else if (use_list) {
                // the groups that hold candidates, in order
                uint32_t c = 0, ng;
                for (int g = g0; g < g1; ++g) c += candidate(top_of(g));
                uint32_t to = block_scan<RW, uint32_t>(c, scan32, ng);
                use_list = ng <= LIST;   // each holds one at least
                if (use_list && c)
                    for (int g = g0; g < g1; ++g)
                        if (candidate(top_of(g))) group_list[to++] = (uint32_t)g;
                __syncthreads();
                // their candidates, in order: a wave a group, its groups consecutive, up to DEEP in flight
                uint32_t m_before = 0;
                constexpr int DEEP = RW == 16 ? 4 : 8;
                const int deep = (int)min((uint32_t)DEEP, (ng + RW - 1) / RW);
                for (uint32_t i0 = 0; use_list && i0 < ng; i0 += RW * deep) {
                    Raw1<T> raw[DEEP];
                    float v[DEEP];
                    int at0[DEEP];
                    uint64_t who[DEEP];
                    uint32_t own = 0;
#pragma unroll
                    for (int o = 0; o < DEEP; ++o) {
                        const uint32_t i = i0 + wave * deep + o;
                        at0[o] = o < deep && i < ng ? (int)group_list[i] * GROUP + lane : n;
                    }
#pragma unroll
                    for (int o = 0; o < DEEP; ++o) raw[o].load(x, mask, at0[o], n);
#pragma unroll
                    for (int o = 0; o < DEEP; ++o) {
                        v[o] = raw[o].value(at0[o], n);
                        who[o] = __ballot(candidate(v[o]));
                        own += (uint32_t)__popcll(who[o]);
                    }
                    if (lane == 0) scan32[wave] = own;
                    __syncthreads();
                    uint32_t owns = lane < RW ? scan32[lane] : 0;
                    owns = wave_scan(owns);
                    uint32_t at = m_before + (wave ? read_lane(owns, wave - 1) : 0);
                    m_before += read_lane(owns, RW - 1);
#pragma unroll
                    for (int o = 0; o < DEEP; ++o) {
                        const uint32_t mine = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(who[o] >> 32),
                                                                             __builtin_amdgcn_mbcnt_lo((uint32_t)who[o], 0));
                        if ((who[o] >> lane & 1) && mine < LIST) {
                            list_key[mine] = key_of(v[o]);
                            list_at[mine] = (uint32_t)at0[o];
                        }
                        at += (uint32_t)__popcll(who[o]);
                    }
                    __syncthreads();
                }
                if (tid == 0) listed = m_before;
            }
        }
        __syncthreads();
        uint32_t m = use_list ? listed : LIST + 1;
        if (m <= 64 && !s.nucleus(n)) {
            // a candidate a lane, in index order: its rank and the mass before it, by every wave over its
            // share of the others, then the answer by one wave's prefix sums
            const bool is = lane < (int)m;
            const uint32_t key = is ? list_key[lane] : 0;
            const double real = is ? W.real(of_key(key)) : 0.0;
            const uint64_t w = is ? W.fixed(real) : 0;
            bool kept = is;
            if (s.k < n) {
                uint32_t rank = 0;
                uint64_t before = 0;
                for (int i = wave; i < (int)m; i += RW) {
                    const uint32_t ki = read_lane(key, i);
                    const bool first = (ki > key) | ((ki == key) & (i < lane));
                    const uint64_t wi = read_lane(w, i);
                    rank += first;
                    before += first ? wi : 0;
                }
                count[tid] = rank;
                mass[tid] = before;
                __syncthreads();
                if (wave != 0) return;
#pragma unroll
                for (int v = 1; v < RW; ++v) {
                    rank += count[v * 64 + lane];
                    before += mass[v * 64 + lane];
                }
                kept = is && rank < (uint32_t)s.k;
                if (s.p < 1.0f) {
                    const double limit = (double)s.p * (double)wave_sum<uint64_t>(kept ? w : 0);
                    kept = kept && (rank == 0 || (double)before < limit);
                }
            }
            if (wave != 0) return;
            const uint64_t own = kept && real >= q ? w : 0, upto = wave_scan(own), sum = last_lane(upto);
            const double t = (double)s.u * (double)sum;
            if (own && (double)upto > t && !((double)(upto - own) > t))   // one lane
                answer(A, r, (int)list_at[lane], real * A.unit / (double)sum);
            return;
        }
        if (!cut && m <= LIST) {
            // min-p alone: prefix sums of the list, by one wave without a barrier
            if (wave != 0) return;
            const uint32_t share = (m + 63) / 64, i0 = min(lane * share, m), i1 = min(i0 + share, m);
            auto kept_weight = [&](uint32_t i) __attribute__((always_inline)) -> uint64_t {
                const double w = W.real(of_key(list_key[i]));
                return w >= q ? W.fixed(w) : 0;
            };
            uint64_t own = 0;
            for (uint32_t i = i0; i < i1; ++i) own += kept_weight(i);
            uint64_t upto = wave_scan(own);
            const uint64_t sum = last_lane(upto);
            const double t = (double)s.u * (double)sum;
            if (own && (double)upto > t && !((double)(upto - own) > t)) {   // one lane
                upto -= own;
                for (uint32_t i = i0; i < i1; ++i) {
                    upto += kept_weight(i);
                    if ((double)upto > t) {
                        answer(A, r, (int)list_at[i], W.real(of_key(list_key[i])) * A.unit / (double)sum);
                        break;
                    }
                }
            }
            return;
        }
        bool from_list = m <= LIST;
        constexpr int PAIRS = 256;
        if (cut && m <= PAIRS) {
            // each candidate's rank and the mass before it, by comparing all pairs: four to sixteen threads
            // a candidate, sixteen bytes of LDS a comparison, no branches (350 cycles a comparison with them)
            constexpr int AT_ONCE = NT / 4, ROUNDS = PAIRS / AT_ONCE;   // candidates a round, of four threads
            const int shift = m * 16 <= NT ? 4 : m * 8 <= NT ? 3 : 2, others = 1 << shift, mine = tid & (others - 1);
            uint4 *const cand = (uint4 *)mass;   // key, index, weight
            if (tid < (int)m) {
                const uint64_t w = W.fixed(W.real(of_key(list_key[tid])));
                cand[tid] = make_uint4(list_key[tid], list_at[tid], (uint32_t)w, (uint32_t)(w >> 32));
            }
            if (tid == 0) {
                found_bin = 0xFFFFFFFFu;
                found_count = 0;
            }
            __syncthreads();
            uint32_t rank[ROUNDS], key[ROUNDS];
            uint64_t before[ROUNDS], s1 = 0;
            bool own[ROUNDS];   // the thread that answers for a candidate
#pragma unroll
            for (int o = 0; o < ROUNDS; ++o) {
                const uint32_t j = o * AT_ONCE + (tid >> shift);
                rank[o] = key[o] = 0;
                before[o] = 0;
                own[o] = mine == 0 && j < m;
                if (o * AT_ONCE >= (int)m) continue;
                const uint4 me = cand[min(j, m - 1)];
                key[o] = me.x;
#pragma unroll 4
                for (uint32_t i = mine; i < m; i += others) {
                    const uint4 c = cand[i];
                    const bool first = (c.x > me.x) | ((c.x == me.x) & (c.y < me.y));
                    rank[o] += first;
                    before[o] += first ? c.z | (uint64_t)c.w << 32 : 0;
                }
                for (int d = 1; d < others; d <<= 1) {
                    rank[o] += __shfl_xor(rank[o], d);
                    before[o] += __shfl_xor(before[o], d);
                }
                s1 += own[o] && rank[o] < (uint32_t)s.k ? me.z | (uint64_t)me.w << 32 : 0;
            }
            double limit = limit_row;
            bool inside = true;
            if (!binned && s.p < 1.0f) {
                s1 = block_sum<RW, uint64_t>(s1, scan64);
                // top-p alone: the list has to hold all of the nucleus
                inside = s.k < n || (double)s1 >= limit_row;
                if (s.k < n) limit = (double)s.p * (double)s1;
            }
            if (inside) {
                bool kept[ROUNDS];
#pragma unroll
                for (int o = 0; o < ROUNDS; ++o) {
                    kept[o] = own[o] && rank[o] < (uint32_t)s.k &&
                              (s.p >= 1.0f || (above_list == 0 && rank[o] == 0) || (double)(above_list + before[o]) < limit);
                    if (kept[o]) atomicMin(&found_bin, key[o]);
                }
                __syncthreads();
                kt = found_bin;
#pragma unroll
                for (int o = 0; o < ROUNDS; ++o)
                    if (kept[o] && key[o] == kt) atomicAdd(&found_count, 1u);
                __syncthreads();
                nt = found_count;
            } else {
                from_list = false;
            }
            __syncthreads();
        }
        // larger cuts: a radix search over the listed candidates or, where they are too many, the row
        auto each = [&](auto &&f) __attribute__((always_inline)) {   // f(x, index) for every candidate, or every entry
            if (from_list) {
                for (uint32_t i = tid; i < m; i += NT) f(of_key(list_key[i]), (int)list_at[i]);
            } else {
                for (int c = wave; c < pieces; c += RW) {
                    float v[8];
                    load8(x, mask, c * PIECE + lane * 8, n, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f(v[e], c * PIECE + lane * 8 + e);
                }
            }
        };
        // the key at which a prefix of the order ends, three levels of a radix search: by count (the
        // prefix has k entries) or by mass (the last entry with less than `limit` before it). From
        // keys >= least, with above_mass over all of them. above_*: of the keys over the found one;
        // count_in: of the found one itself.
        uint64_t above_mass = 0, all_mass = 0;
        uint32_t above_count = 0, count_in = 0;
        bool found = true;   // false: by count, and there are no more than k entries; all_mass is theirs
        auto search = [&](bool by_mass, bool with_mass, uint32_t least, uint32_t k, double limit) __attribute__((always_inline)) {
            uint32_t prefix = 0;
            above_count = 0;
            for (int level = 0; level < 3; ++level) {
                const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
#pragma unroll
                for (int b = 0; b < BT; ++b) {
                    mass[b * NT + tid] = 0;
                    count[b * NT + tid] = 0;
                }
                __syncthreads();
                each([&](float v, int) __attribute__((always_inline)) {
                    const uint32_t key = key_of(v);
                    if (key == 0 || key < least || (level > 0 && key >> (shift + bits) != prefix)) return;
                    const uint32_t b = (key >> shift) & ((1u << bits) - 1);
                    atomicAdd(&count[b], 1u);
                    if (with_mass) atomicAdd((unsigned long long *)&mass[b], (unsigned long long)W.fixed(W.real(v)));
                });
                __syncthreads();
                // bins from the top, BT a thread
                uint64_t m_sum = 0, m_all;
                uint32_t c_sum = 0, c_all;
#pragma unroll
                for (int b = 0; b < BT; ++b) {
                    m_sum += mass[BINS - 1 - tid * BT - b];
                    c_sum += count[BINS - 1 - tid * BT - b];
                }
                uint64_t m_ex = above_mass + block_scan<RW, uint64_t>(m_sum, scan64, m_all);
                uint32_t c_ex = above_count + block_scan<RW, uint32_t>(c_sum, scan32, c_all);
                if (!by_mass && level == 0 && c_all <= k) {   // for all threads
                    found = false;
                    all_mass = m_all;
                    __syncthreads();
                    return 0u;
                }
#pragma unroll
                for (int b = 0; b < BT; ++b) {
                    const int at = BINS - 1 - tid * BT - b;
                    const uint64_t m_in = m_ex + mass[at];
                    const uint32_t c_in = c_ex + count[at];
                    const bool here = by_mass ? (m_ex == 0 || (double)m_ex < limit) && (double)m_in >= limit && m_in > m_ex
                                              : c_ex < k && c_in >= k;
                    if (here) {   // one bin of one thread
                        found_bin = (uint32_t)at;
                        found_mass = m_ex;
                        found_count = c_ex;
                    }
                    m_ex = m_in;
                    c_ex = c_in;
                }
                __syncthreads();
                const uint32_t b = found_bin & (BINS - 1);
                above_mass = found_mass;
                above_count = found_count;
                count_in = count[b];
                prefix = (prefix << bits) | b;
                __syncthreads();
            }
            return prefix;
        };
        auto mass_of_all = [&]() __attribute__((always_inline)) {
            uint64_t w = 0;
            each([&](float v, int) __attribute__((always_inline)) {
                if (v != -INFINITY) w += W.fixed(W.real(v));
            });
            return block_sum<RW, uint64_t>(w, scan64);
        };
        if (W.hard && s.greedy) {
            kt = key_of(top);
            nt = 1;
        } else if (cut && kt == 0) {
            uint64_t s1 = 0;
            bool k_cut = false;
            if (s.k < n) {
                kt = search(false, s.p < 1.0f, 0, (uint32_t)s.k, 0.0);
                k_cut = found;
                if (k_cut) {
                    nt = (uint32_t)s.k - above_count;
                    s1 = above_mass + nt * W.fixed(W.real(of_key(kt)));
                } else {
                    s1 = all_mass;
                }
            } else {
                s1 = mass_of_all();
                if (from_list && !binned && (double)s1 < limit_row) {   // the nucleus is not inside the list
                    from_list = false;
                    s1 = mass_of_all();
                }
            }
            if (s.p < 1.0f) {
                // with a list, the entries behind it count in the limit only
                const double limit = from_list && s.k == n ? limit_row : (double)s.p * (double)s1;
                if (limit <= 0.0) {
                    kt = key_of(top);
                    nt = 1;
                } else {
                    const uint32_t kk = kt, kn = nt;
                    above_mass = from_list ? above_list : 0;
                    kt = search(true, true, kk, 0, limit);
                    // tie j stays while above + j w < limit
                    const uint64_t w = W.fixed(W.real(of_key(kt)));
                    const double more = w ? ceil((limit - (double)above_mass) / (double)w) : (double)count_in;
                    nt = (uint32_t)fmin(fmax(more, 1.0), (double)count_in);
                    if (k_cut && kt == kk) nt = min(nt, kn);
                }
            }
        }
        const bool bounded = kt != 0;

        if (from_list && !binned) {
            // the list is in index order and holds all that is kept: its prefix sums answer
            const uint32_t share = (m + NT - 1) / NT, i0 = min(tid * share, m), i1 = min(i0 + share, m);
            uint32_t t = 0, all_ties;
            for (uint32_t i = i0; i < i1; ++i) t += bounded && list_key[i] == kt;
            uint32_t rank = block_scan<RW, uint32_t>(t, scan32, all_ties);
            const uint32_t rank0 = rank;
            auto kept_weight = [&](uint32_t i) __attribute__((always_inline)) -> uint64_t {
                const uint32_t key = list_key[i];
                if (key < kt || (bounded && key == kt && rank++ >= nt)) return 0;
                const double w = W.real(of_key(key));
                return w >= q ? W.fixed(w) : 0;
            };
            uint64_t own = 0, sum;
            for (uint32_t i = i0; i < i1; ++i) own += kept_weight(i);
            uint64_t upto = block_scan<RW, uint64_t>(own, scan64, sum);
            const double t_sum = (double)s.u * (double)sum;
            if (own && !((double)upto > t_sum) && (double)(upto + own) > t_sum) {   // one thread
                rank = rank0;
                for (uint32_t i = i0; i < i1; ++i) {
                    upto += kept_weight(i);
                    if ((double)upto > t_sum) {
                        answer(A, r, (int)list_at[i], W.real(of_key(list_key[i])) * A.unit / (double)sum);
                        break;
                    }
                }
            }
            return;
        }

        // masses and ties by segment, in index order
        const double wt = bounded ? W.real(of_key(kt)) : 0.0;
        const uint64_t wtie = wt >= q ? W.fixed(wt) : 0;
        if (from_list) {
            seg_mass[tid] = binned ? kept_above : 0;
            seg_ties[tid] = 0;
            __syncthreads();
            each([&](float v, int i) __attribute__((always_inline)) {
                const uint32_t key = key_of(v);
                const int g = i / (PIECE * REC) / per;
                if (key > kt) {
                    const double wr = W.real(v);
                    if (wr >= q) atomicAdd((unsigned long long *)&seg_mass[g], (unsigned long long)W.fixed(wr));
                } else if (bounded && key == kt) {
                    atomicAdd(&seg_ties[g], 1u);
                }
            });
        } else {
            __syncthreads();
            for (int g = wave; g < segs; g += RW) {
                uint64_t w_sum = 0, t_sum = 0;
                for (int c = g * per * REC; c < min((g + 1) * per * REC, pieces); ++c) {
                    float v[8];
                    load8(x, mask, c * PIECE + lane * 8, n, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t key = key_of(v[e]);
                        if (key > kt) {
                            const double w = W.real(v[e]);
                            w_sum += w >= q ? W.fixed(w) : 0;
                        }
                        t_sum += bounded && key == kt;
                    }
                }
                w_sum = wave_sum(w_sum);
                t_sum = wave_sum(t_sum);
                if (lane == 0) {
                    seg_mass[g] = w_sum;
                    seg_ties[g] = (uint32_t)t_sum;
                }
            }
        }
        __syncthreads();
        const uint32_t mine = tid < segs ? seg_ties[tid] : 0;
        uint32_t all_ties;
        const uint32_t ties_ex = block_scan<RW, uint32_t>(mine, scan32, all_ties);
        const uint32_t left = nt > ties_ex ? nt - ties_ex : 0;
        const uint64_t here = (tid < segs ? seg_mass[tid] : 0) + (uint64_t)min(mine, left) * wtie;
        uint64_t sum;
        const uint64_t m_ex = block_scan<RW, uint64_t>(here, scan64, sum);
        target = (double)s.u * (double)sum;
        scale_out = A.unit / (double)sum;
        if ((double)(m_ex + here) > target && !((double)m_ex > target)) {   // one thread
            found_bin = (uint32_t)tid;
            found_mass = m_ex;
            found_count = ties_ex;
        }
        __syncthreads();
        seg = (int)found_bin;
        base = found_mass;
        ties = found_count;
    }
    // inside the segment: four waves, a piece each
    const int first = seg * per * REC, end = min((seg + 1) * per * REC, pieces);
    if (plain) {
        // rounding may leave the target just over the segment's end: the next entry that weighs half a
        // unit then, or the row's last one; if all from the segment on are lighter, the row's first
        int last = -1;
        float xl = 0.0f;
        for (int c0 = first;; c0 += 4) {
            if (c0 >= pieces) {
                if (last >= 0) break;
                c0 = 0;
                target = -1.0;
            }
            const int c = c0 + wave, i = c * PIECE + lane * 8;
            double w8[8], own = 0.0, in = 0.0;
            float v[8], xm = 0.0f;
            int mine = -1;
            const bool works = wave < 4 && c < pieces;
            if (works) {
                load8(x, mask, i, n, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w8[e] = W.real(v[e]);
                    w8[e] = v[e] != -INFINITY && W.fixed(w8[e]) ? w8[e] : 0.0;
                    own += w8[e];
                    if (w8[e] > 0.0) {
                        mine = i + e;
                        xm = v[e];
                    }
                }
                in = wave_scan(own);
            }
            const uint64_t some = __ballot(mine >= 0);
            const int who = some ? 63 - __clzll((long long)some) : 0;
            mine = __builtin_amdgcn_readlane(mine, who);
            xm = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(xm), who));
            if (wave < 4 && lane == 63) {
                final_sum[wave] = in;
                final_last[wave] = some ? mine : -1;
                final_x[wave] = xm;
            }
            __syncthreads();
            double upto = base_real;
#pragma unroll
            for (int w = 0; w < 4; ++w) upto += w < wave ? final_sum[w] : 0.0;
            upto += in - own;
            int at = -1;
            float xa = 0.0f;
            if (works) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    upto += w8[e];
                    if (at < 0 && w8[e] > 0.0 && upto > target) {
                        at = i + e;
                        xa = v[e];
                    }
                }
            }
            const uint64_t hits = __ballot(at >= 0);
            if (wave < 4 && lane == 0) final_hit[wave] = hits ? 1 : 0;
            __syncthreads();
            int by = -1;
#pragma unroll
            for (int w = 3; w >= 0; --w) by = final_hit[w] ? w : by;
            if (by >= 0) {
                if (wave == by && lane == __ffsll((unsigned long long)hits) - 1) answer(A, r, at, W.real(xa) * scale_out);
                return;
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                base_real += final_sum[w];
                if (final_last[w] >= 0) {
                    last = final_last[w];
                    xl = final_x[w];
                }
            }
            __syncthreads();
        }
        if (tid == 0) answer(A, r, last, W.real(xl) * scale_out);
        return;
    }
    const bool bounded = kt != 0;
    const double wt = bounded ? W.real(of_key(kt)) : 0.0;
    const uint64_t wtie = wt >= q ? W.fixed(wt) : 0;
    for (int c0 = first; c0 < end; c0 += 4) {
        const int c = c0 + wave, i = c * PIECE + lane * 8;
        const bool works = wave < 4 && c < end;
        float v[8];
        uint32_t t = 0;
        if (works) {
            load8(x, mask, i, n, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) t += bounded && key_of(v[e]) == kt;
        }
        const uint32_t t_in = wave_scan(t);
        if (wave < 4 && lane == 63) final_ties[wave] = t_in;
        __syncthreads();
        uint32_t rank = ties + t_in - t;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            rank += w < wave ? final_ties[w] : 0;
            ties += final_ties[w];
        }
        uint64_t w8[8], own = 0;
        if (works) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t key = key_of(v[e]);
                w8[e] = 0;
                if (key > kt) {
                    const double w = W.real(v[e]);
                    w8[e] = w >= q ? W.fixed(w) : 0;
                } else if (bounded && key == kt) {
                    w8[e] = rank++ < nt ? wtie : 0;
                }
                own += w8[e];
            }
        }
        const uint64_t in = wave_scan(own);
        if (wave < 4 && lane == 63) final_mass[wave] = in;
        __syncthreads();
        uint64_t upto = base + in - own;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            upto += w < wave ? final_mass[w] : 0;
            base += final_mass[w];
        }
        if (works && !((double)upto > target) && (double)(upto + own) > target) {   // one thread of the row's
            int at = -1;
            float xa = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                upto += w8[e];
                if (at < 0 && w8[e] && (double)upto > target) {
                    at = i + e;
                    xa = v[e];
                }
            }
            answer(A, r, at, W.real(xa) * scale_out);
        }
        if ((double)base > target) return;   // answered
    }
}

// ---------------------------------------------------------------- launches
// Rows up to here are held in registers: sixteen entries a lane of four waves. Twice that, sixteen waves
// (8,192 fp32, 8 rows): 20 us top-k 40 and 35 top-p 0.9, against 12 and 33 by the groups' maxima.
constexpr int WAVE_N = 4096;
constexpr int64_t GRID = 1 << 22;    // rows of one launch: the card's grids end at 2^32 threads
// A CU holds one row's workgroup of 16 waves, two of 8 or four of 4; more rows than 256 CUs hold at once
// take smaller ones. bf16 rows of 16,384: 511 rows, top-k 40, 13.6 us by 8 waves each and 14.9 by 16, whole
// 16.1 and 17.9; 1,000 rows 19.6 by 4 and 23.5 by 8, whole 23.1 and 27.7 (min-p over longer rows loses a
// tenth: 640 rows of 32,000 34 and 31).
constexpr int64_t ROWS_OF_16 = 256, ROWS_OF_8 = 512;
// From here on rows of 513 to 1,024 entries take one wave instead of four: bf16, top-p 0.9, 4,096 rows
// 26 us against 45, 1,024 rows 14 against 17, 511 rows 14 against 12.
constexpr int64_t ONE_WAVE_FROM = 768;
// rows whose workgroup scans them itself: a piece a wave
static bool fused(int64_t rows, int64_t n) { return rows <= ROWS_OF_16 && n <= 16 * PIECE; }

// the workspace's parts, in bytes from its start
struct SampleSpace {
    int blocks = 0, splits = 0;
    int64_t chunk = 0;   // rows of a launch of the nucleus kernels
    int64_t masses = 0, block_tops = 0, tops = 0, bins = 0, kept = 0, lists = 0, listed = 0, heads = 0, bytes = 0;
    SampleSpace(int64_t rows, int64_t n) {
        if (n <= WAVE_N || fused(rows, n) || rows == 0) return;
        blocks = ceil_div(n, BLOCK);
        splits = (int)std::max<int64_t>(1, std::min<int64_t>({SPLITS, 1024 / rows, (blocks + 3) / 4}));
        chunk = std::min<int64_t>(rows, 2048 / splits);
        auto take = [&](int64_t size) {
            const int64_t at = bytes;
            bytes += (size + 15) / 16 * 16;
            return at;
        };
        masses = take(rows * blocks * 8);
        block_tops = take(rows * blocks * 4);
        tops = take(rows * blocks * BP * GP * 4);
        bins = take(chunk * splits * NBINS * 8);
        kept = take(chunk * blocks * 8);
        lists = take(chunk * splits * NLIST * 8);
        listed = take(chunk * splits * 4);
        heads = take(chunk * (int64_t)sizeof(SampleHead));
    }
};

static void check_shape(int64_t rows, int64_t n) {
    SNK_CHECK(rows >= 0 && rows < (int64_t)1 << 31, SNK_ERR_INVALID, "sample: %lld rows", (long long)rows);
    SNK_CHECK(n >= 1 && n <= 1 << 24, SNK_ERR_INVALID, "sample: %lld logits a row, 1 to 2^24 are supported", (long long)n);
}

static SampleArgs sample_args(const snk_sample_cfg_t *cfg, int64_t rows, int64_t n) {
    SNK_CHECK(cfg, SNK_ERR_INVALID, "sample: cfg is NULL");
    SNK_CHECK(cfg->struct_size == (int32_t)sizeof(snk_sample_cfg_t), SNK_ERR_INVALID,
              "snk_sample_cfg_t.struct_size = %d, the library's struct has %d bytes (binding out of date)",
              cfg->struct_size, (int)sizeof(snk_sample_cfg_t));
    SNK_CHECK(cfg->dtype == SNK_F32 || cfg->dtype == SNK_BF16 || cfg->dtype == SNK_F16, SNK_ERR_INVALID,
              "sample: unknown element type %d", cfg->dtype);
    check_shape(rows, n);
    SNK_CHECK(cfg->temperature >= 0 && cfg->temperature < INFINITY, SNK_ERR_INVALID, "sample: temperature %g",
              cfg->temperature);
    SNK_CHECK(cfg->top_k >= 0, SNK_ERR_INVALID, "sample: top_k %d is negative", cfg->top_k);
    SNK_CHECK(cfg->top_p >= 0 && cfg->top_p <= 1, SNK_ERR_INVALID, "sample: top_p %g outside [0, 1]", cfg->top_p);
    SNK_CHECK(cfg->min_p >= 0 && cfg->min_p <= 1, SNK_ERR_INVALID, "sample: min_p %g outside [0, 1]", cfg->min_p);
    SampleArgs A{};
    A.rows = rows;
    A.n = (int32_t)n;
    A.temperature = cfg->temperature;
    A.top_k = cfg->top_k;
    A.top_p = cfg->top_p;
    A.min_p = cfg->min_p;
    A.t_dev = cfg->temperature_dev;
    A.k_dev = cfg->top_k_dev;
    A.p_dev = cfg->top_p_dev;
    A.q_dev = cfg->min_p_dev;
    int log2n = 0;
    while (((int64_t)1 << log2n) < n) ++log2n;
    A.unit = std::ldexp(1.0, std::min(51, 61 - log2n));
    return A;
}

template <class T>
static void sample_launch_t(SampleArgs A, uint8_t *ws, hipStream_t s) {
    if (A.n <= 8) {
        const unsigned few = (unsigned)ceil_div(A.rows, 256);
        if (A.n <= 4)
            sample_few_kernel<T, 4><<<few, 256, 0, s>>>(A);
        else
            sample_few_kernel<T, 8><<<few, 256, 0, s>>>(A);
        launch_check("sample_few_kernel");
        return;
    }
    const bool many = A.rows > ROWS_OF_16;
    // a top-k that the groups' maxima bound, so that its candidates are few: 8 rows of 4,096, top-k 40,
    // 11 us against 15, with top-p 0.9 11 against 17. Not for more rows, which that path scans into a
    // workspace: rows of up to 4,096 entries need none. It costs them time (4,096 rows of 4,096 bf16, top-k
    // 40, 68 us here, rows of 8,192 by the maxima 52; 65,536 rows 980 and 815).
    const bool by_groups = !many && A.n > 2048 && !A.k_dev && A.top_k > 0 && A.top_k <= A.n / GROUP;
    if (A.n <= WAVE_N && !by_groups) {
        for (; A.row0 < A.rows; A.row0 += GRID) {
            const unsigned rows = (unsigned)std::min(GRID, A.rows - A.row0), fours = (rows + 3) / 4;
            if (A.n <= 64)
                sample_wave_kernel<T, 1, 1><<<fours, 256, 0, s>>>(A);
            else if (A.n <= 128)
                sample_wave_kernel<T, 2, 1><<<fours, 256, 0, s>>>(A);
            else if (A.n <= 256)
                sample_wave_kernel<T, 4, 1><<<fours, 256, 0, s>>>(A);
            else if (A.n <= 512)
                sample_wave_kernel<T, 8, 1><<<fours, 256, 0, s>>>(A);
            else if (A.n <= 1024 && A.rows >= ONE_WAVE_FROM)
                sample_wave_kernel<T, 16, 1><<<fours, 256, 0, s>>>(A);
            else if (A.n <= 1024)
                sample_wave_kernel<T, 4, 4><<<rows, 256, 0, s>>>(A);
            else if (A.n <= 2048)
                sample_wave_kernel<T, 8, 4><<<rows, 256, 0, s>>>(A);
            else
                sample_wave_kernel<T, 16, 4><<<rows, 256, 0, s>>>(A);
            launch_check("sample_wave_kernel");
        }
        return;
    }
    const bool nucleus = (A.p_dev || A.top_p < 1.0f) && (A.k_dev || A.top_k == 0 || A.top_k >= A.n);
    if constexpr (sizeof(T) == 2)
        if (fused(A.rows, A.n) && nucleus && !A.k_dev) {
            // top-p alone has no bound by the groups: in the registers of sixteen waves, 128 rows of 8,192
            // bf16 23 us against 34, fp16 25 (fp32's keys have twice the bits: 37 against 34)
            sample_wave_kernel<T, 8, 16><<<(unsigned)A.rows, 1024, 0, s>>>(A);
            launch_check("sample_wave_kernel");
            return;
        }
    if (fused(A.rows, A.n)) {
        sample_row_kernel<T, 16, 1><<<(unsigned)A.rows, 1024, 0, s>>>(A);
        launch_check("sample_row_kernel");
        return;
    }
    // up to 32,768, four pieces a wave, where top-p alone does not need its passes over the scan's
    // records: 8 bf16 rows of 16,384, top-k 40, 10.7 us against 12.7 with the scan's own launch, 256 rows
    // of 32,000 10.1 against 12.8
    if (!many && A.n <= 16 * BLOCK && !nucleus) {
        sample_row_kernel<T, 16, BP><<<(unsigned)A.rows, 1024, 0, s>>>(A);
        launch_check("sample_row_kernel");
        return;
    }
    const SampleSpace S(A.rows, A.n);
    A.masses = (double *)(ws + S.masses);
    A.block_tops = (float *)(ws + S.block_tops);
    A.tops = (float *)(ws + S.tops);
    const int64_t total = A.rows * S.blocks;
    sample_scan_kernel<T><<<(unsigned)std::min<int64_t>((total + 3) / 4, 4096), 256, 0, s>>>(A, S.blocks, total);
    launch_check("sample_scan_kernel");
    if (nucleus) {
        A.splits = S.splits;
        A.bins = (uint64_t *)(ws + S.bins);
        A.kept = (uint64_t *)(ws + S.kept);
        A.lists = (uint2 *)(ws + S.lists);
        A.listed = (uint32_t *)(ws + S.listed);
        A.heads = (SampleHead *)(ws + S.heads);
    }
    const int64_t chunk = nucleus ? S.chunk : GRID;
    for (; A.row0 < A.rows; A.row0 += chunk) {
        const unsigned rows = (unsigned)std::min(chunk, A.rows - A.row0);
        if (nucleus) {
            sample_bins_kernel<T><<<rows * S.splits, NTH, 0, s>>>(A, S.blocks);
            launch_check("sample_bins_kernel");
            sample_kept_kernel<T><<<rows * S.splits, NTH, 0, s>>>(A, S.blocks);
            launch_check("sample_kept_kernel");
        }
        if (A.rows > ROWS_OF_8)
            sample_row_kernel<T, 4, 0><<<rows, 256, 0, s>>>(A);
        else if (many)
            sample_row_kernel<T, 8, 0><<<rows, 512, 0, s>>>(A);
        else
            sample_row_kernel<T, 16, 0><<<rows, 1024, 0, s>>>(A);
        launch_check("sample_row_kernel");
    }
}

static void sample_launch(const SampleArgs &A, int32_t dtype, void *ws, hipStream_t s) {
    if (A.rows == 0) return;
    if (dtype == SNK_F32)
        sample_launch_t<float>(A, (uint8_t *)ws, s);
    else if (dtype == SNK_BF16)
        sample_launch_t<__bf16>(A, (uint8_t *)ws, s);
    else
        sample_launch_t<_Float16>(A, (uint8_t *)ws, s);
}

}  // namespace snk

using namespace snk;

extern "C" int snk_sample_workspace(int64_t rows, int64_t n, int64_t *bytes) {
    return guard([&] {
        SNK_CHECK(bytes, SNK_ERR_INVALID, "sample_workspace: NULL argument");
        check_shape(rows, n);
        *bytes = SampleSpace(rows, n).bytes;
    });
}

extern "C" int snk_sample_logits(const void *logits, int64_t rows, int64_t n, int64_t ld, const uint8_t *mask,
                                 int64_t ld_mask, const float *u, const snk_sample_cfg_t *cfg, int32_t *idx, float *prob,
                                 void *ws, int64_t ws_bytes) {
    return guard([&] {
        SampleArgs A = sample_args(cfg, rows, n);
        if (rows == 0) return;
        SNK_CHECK(logits && u && idx, SNK_ERR_INVALID, "sample: NULL argument");
        SNK_CHECK(ld == 0 || ld >= n, SNK_ERR_INVALID, "sample: ld %lld of rows of %lld", (long long)ld, (long long)n);
        SNK_CHECK(!mask || ld_mask == 0 || ld_mask >= n, SNK_ERR_INVALID, "sample: ld_mask %lld of rows of %lld",
                  (long long)ld_mask, (long long)n);
        const uintptr_t a = reinterpret_cast<uintptr_t>(logits);
        SNK_CHECK(a % (cfg->dtype == SNK_F32 ? 4 : 2) == 0, SNK_ERR_INVALID, "sample: logits are not element-aligned");
        int64_t need = 0;
        if (snk_sample_workspace(rows, n, &need) != SNK_OK) throw Error{SNK_ERR_INVALID};
        SNK_CHECK(need == 0 || (ws && ws_bytes >= need && reinterpret_cast<uintptr_t>(ws) % 16 == 0), SNK_ERR_INVALID,
                  "sample: a 16-byte aligned workspace of %lld bytes is needed, %lld given", (long long)need,
                  (long long)(ws ? ws_bytes : 0));
        A.x = logits;
        A.ld = ld;
        A.mask = mask;
        A.ld_mask = ld_mask;
        A.u = u;
        A.idx = idx;
        A.prob = prob;
        sample_launch(A, cfg->dtype, ws, stream());
    });
}

extern "C" int snk_dqn_act_sample(snk_dqn h, snk_env env, const snk_sample_cfg_t *cfg, uint64_t seed, uint8_t *act) {
    return guard([&] {
        SNK_CHECK(h && env && act, SNK_ERR_INVALID, "NULL argument");
        const EnvDev &E = env_dev(env);
        SNK_CHECK(E.bs == h->L.bs && E.C == h->L.C, SNK_ERR_INVALID, "env/model geometry mismatch");
        SampleArgs A = sample_args(cfg, E.n, 3);
        SNK_CHECK(cfg->dtype == SNK_F32, SNK_ERR_INVALID, "act_sample: Q values are fp32");
        hipStream_t s = stream();
        A.x = dqn_q_env(h, SNK_NET_Q, env, s);
        A.ld = 3;
        A.act = act;
        A.seed = seed;
        A.tptr = &E.ctl->t;
        sample_launch(A, SNK_F32, nullptr, s);   // 3 entries a row: no workspace
    });
}
