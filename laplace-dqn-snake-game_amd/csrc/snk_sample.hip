// snk_sample.hip — one index a row from logits: temperature, top-k, top-p, min-p and a given random
// number (include/snakehip.h states the rules).
//
// Every filter keeps a prefix of the order (x descending, equal ones by lower index), so a row's
// answer needs no sort: the prefix is a cut (key kt, nt): the entries above kt and the first nt of
// the entries equal to it, in index order. Masses are integers (weights rounded to 2^-sh of the
// largest), so sums in LDS atomics and over any split of the row are exact and always the same.
#include <algorithm>
#include <cmath>

#include "snk_dqn.hpp"

namespace snk {

constexpr int PIECE = 512;      // consecutive elements a wave reads at once: 8 a lane
constexpr int BINS = 2048;      // of a level of the radix search: 11 + 11 + 10 bits of the key

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
};

// a row's settings, the same for all its threads
struct SampleRow {
    double inv_t;
    bool greedy;
    int k;        // 1..n
    float p, q, u;
};
__device__ __forceinline__ SampleRow sample_row(const SampleArgs &A, int64_t r) {
    SampleRow s;
    const float t = A.t_dev ? A.t_dev[r] : A.temperature;
    s.greedy = !(t > 0.0f);
    s.inv_t = s.greedy ? 0.0 : 1.0 / (double)t;
    const int k = A.k_dev ? A.k_dev[r] : A.top_k;
    s.k = s.greedy ? 1 : k > 0 && k < A.n ? k : A.n;
    const float p = A.p_dev ? A.p_dev[r] : A.top_p, q = A.q_dev ? A.q_dev[r] : A.min_p;
    s.p = p < 1.0f ? fmaxf(p, 0.0f) : 1.0f;   // NaN: off
    s.q = q > 0.0f ? fminf(q, 1.0f) : 0.0f;
    const float u = A.u ? A.u[r] : rng_uniform(rng_hash(A.seed, (uint64_t)r, (uint64_t)*A.tptr));
    s.u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    return s;
}

// order-preserving key of an allowed logit; 0 for -inf (excluded)
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return x == -INFINITY ? 0u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

struct Weight {
    double top, inv_t, unit;
    bool hard;   // only entries equal to the largest weigh: temperature 0, or +inf among them
    __device__ __forceinline__ double real(float x) const {
        if (hard) return (double)x == top ? 1.0 : 0.0;
        return exp(((double)x - top) * inv_t);
    }
    __device__ __forceinline__ uint64_t fixed(double w) const { return (uint64_t)rint(w * unit); }
};

template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) pack8 {
    T v[8];
};
// elements i..i+7 of a row, -inf where masked or behind the end; -0 becomes +0 (they are equal)
template <class T>
__device__ __forceinline__ void load8(const T *x, const uint8_t *mask, int i, int n, float *v) {
    if (i + 8 <= n) {
        const pack8<T> q = *reinterpret_cast<const pack8<T> *>(x + i);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)q.v[k] + 0.0f;
        if (mask) {
            const pack8<uint8_t> m = *reinterpret_cast<const pack8<uint8_t> *>(mask + i);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = m.v[k] ? -INFINITY : v[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            v[k] = i + k < n && !(mask && mask[i + k]) ? (float)x[i + k] + 0.0f : -INFINITY;
    }
}

template <class V>
__device__ __forceinline__ V wave_scan(V v, int lane) {   // inclusive
    for (int o = 1; o < 64; o <<= 1) {
        const V y = __shfl_up(v, o);
        if (lane >= o) v += y;
    }
    return v;
}
template <class V>
__device__ __forceinline__ V wave_sum(V v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

__device__ __forceinline__ void answer(const SampleArgs &A, int64_t r, int i, double prob) {
    if (A.act) {
        A.act[r] = (uint8_t)(i < 0 ? 0 : i);
        return;
    }
    A.idx[r] = i;
    if (A.prob) A.prob[r] = (float)prob;
}

// ---------------------------------------------------------------- a thread a row: n <= N
template <class T, int N>
__global__ __launch_bounds__(256) void sample_few_kernel(SampleArgs A) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= A.rows) return;
    const SampleRow s = sample_row(A, r);
    const T *x = (const T *)A.x + r * A.ld;
    const uint8_t *mask = A.mask ? A.mask + r * A.ld_mask : nullptr;
    float v[N], top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = i < A.n && !(mask && mask[i]) ? (float)x[i] + 0.0f : -INFINITY;
        nan |= v[i] != v[i];
        top = fmaxf(top, v[i]);
    }
    if (nan || top == -INFINITY) {
        answer(A, r, -1, nan ? NAN : 0.0);
        return;
    }
    const Weight W{(double)top, s.inv_t, A.unit, s.greedy || top == INFINITY};
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

// ---------------------------------------------------------------- a workgroup a row
constexpr int RW = 16;          // waves
constexpr int SEGS = 1024;      // most segments the row's masses are kept by

// exclusive prefix of v over the workgroup's threads; total: of all. sh: RW + 1 values
template <class V>
__device__ __forceinline__ V block_scan(V v, V *sh, V &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const V in = wave_scan(v, lane);
    __syncthreads();
    if (lane == 63) sh[wave] = in;
    __syncthreads();
    if (wave == 0) {
        const V x = lane < RW ? sh[lane] : 0;
        const V y = wave_scan(x, lane);
        if (lane < RW) sh[lane] = y - x;
        if (lane == RW - 1) sh[RW] = y;
    }
    __syncthreads();
    total = sh[RW];
    return sh[wave] + in - v;
}

template <class T>
__global__ __launch_bounds__(1024) void sample_row_kernel(SampleArgs A) {
    __shared__ uint64_t mass[BINS];
    __shared__ uint32_t count[BINS];
    __shared__ uint64_t seg_mass[SEGS];
    __shared__ uint32_t seg_ties[SEGS];
    __shared__ uint64_t scan64[RW + 1];
    __shared__ uint32_t scan32[RW + 1];
    __shared__ float wave_top[RW];
    __shared__ int wave_nan[RW];
    __shared__ uint64_t found_mass;
    __shared__ uint32_t found_bin, found_count;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = A.n;
    const SampleRow s = sample_row(A, r);
    const T *x = (const T *)A.x + r * A.ld;
    const uint8_t *mask = A.mask ? A.mask + r * A.ld_mask : nullptr;
    const int pieces = (n + PIECE - 1) / PIECE;

    float top = -INFINITY;
    bool nan = false;
    for (int c = wave; c < pieces; c += RW) {
        float v[8];
        load8(x, mask, c * PIECE + lane * 8, n, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            nan |= v[e] != v[e];
            top = fmaxf(top, v[e]);
        }
    }
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    nan = __ballot(nan) != 0;
    if (lane == 0) {
        wave_top[wave] = top;
        wave_nan[wave] = nan;
    }
    __syncthreads();
    for (int w = 0; w < RW; ++w) {
        top = fmaxf(top, wave_top[w]);
        nan |= wave_nan[w] != 0;
    }
    if (nan || top == -INFINITY) {   // the whole workgroup
        if (tid == 0) answer(A, r, -1, nan ? NAN : 0.0);
        return;
    }
    const Weight W{(double)top, s.inv_t, A.unit, s.greedy || top == INFINITY};

    // the cut: keys above kt, and the first nt of those equal to it
    uint32_t kt = 0, nt = 0;
    // the key at which a prefix of the order ends, three levels of a radix search: by count (the
    // prefix has k entries) or by mass (the last entry with less than `limit` before it). From
    // keys >= least. above_*: of the keys over the found one; count_in: of the found one itself.
    uint64_t above_mass = 0;
    uint32_t above_count = 0, count_in = 0;
    auto search = [&](bool by_mass, bool with_mass, uint32_t least, uint32_t k, double limit) {
        uint32_t prefix = 0;
        above_mass = 0;
        above_count = 0;
        for (int level = 0; level < 3; ++level) {
            const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
            for (int b = tid; b < BINS; b += 1024) {
                mass[b] = 0;
                count[b] = 0;
            }
            __syncthreads();
            for (int c = wave; c < pieces; c += RW) {
                float v[8];
                load8(x, mask, c * PIECE + lane * 8, n, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t key = key_of(v[e]);
                    if (key == 0 || key < least || (level > 0 && key >> (shift + bits) != prefix)) continue;
                    const uint32_t b = (key >> shift) & ((1u << bits) - 1);
                    atomicAdd(&count[b], 1u);
                    if (with_mass)
                        atomicAdd((unsigned long long *)&mass[b], (unsigned long long)W.fixed(W.real(v[e])));
                }
            }
            __syncthreads();
            // bins from the top, two a thread
            const int b0 = BINS - 1 - 2 * tid, b1 = b0 - 1;
            const uint64_t m0 = mass[b0], m1 = mass[b1];
            const uint32_t c0 = count[b0], c1 = count[b1];
            uint64_t m_all;
            uint32_t c_all;
            const uint64_t m_ex = above_mass + block_scan<uint64_t>(m0 + m1, scan64, m_all);
            const uint32_t c_ex = above_count + block_scan<uint32_t>(c0 + c1, scan32, c_all);
            auto test = [&](int b, uint64_t m, uint32_t c, uint64_t mb, uint32_t cb) {
                const bool here = by_mass ? (double)mb < limit && (double)(mb + m) >= limit : cb < k && cb + c >= k;
                if (here) {   // one bin of one thread
                    found_bin = (uint32_t)b;
                    found_mass = mb;
                    found_count = cb;
                }
            };
            test(b0, m0, c0, m_ex, c_ex);
            test(b1, m1, c1, m_ex + m0, c_ex + c0);
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
    const bool nucleus = s.p < 1.0f && !s.greedy;
    uint64_t s1 = 0;
    if (s.greedy) {
        kt = key_of(top);
        nt = 1;
    } else {
        bool whole = true;   // no top-k cut
        if (s.k < n) {
            // fewer allowed entries than k: nothing to cut
            uint32_t allowed = 0;
            for (int c = wave; c < pieces; c += RW) {
                float v[8];
                load8(x, mask, c * PIECE + lane * 8, n, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) allowed += v[e] != -INFINITY;
            }
            uint32_t all;
            block_scan<uint32_t>(allowed, scan32, all);
            if (all > (uint32_t)s.k) {
                kt = search(false, nucleus, 0, (uint32_t)s.k, 0.0);
                nt = (uint32_t)s.k - above_count;
                s1 = above_mass + nt * W.fixed(W.real(of_key(kt)));
                whole = false;
            }
        }
        if (nucleus) {
            if (whole) {
                uint64_t part = 0;
                for (int c = wave; c < pieces; c += RW) {
                    float v[8];
                    load8(x, mask, c * PIECE + lane * 8, n, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (v[e] != -INFINITY) part += W.fixed(W.real(v[e]));
                }
                block_scan<uint64_t>(part, scan64, s1);
            }
            const double limit = (double)s.p * (double)s1;
            if (limit <= 0.0) {
                kt = key_of(top);
                nt = 1;
            } else {
                const uint32_t kk = kt, kn = nt;
                kt = search(true, true, kk, 0, limit);
                // tie j stays while above + j w < limit
                const uint64_t w = W.fixed(W.real(of_key(kt)));
                const double more = w ? ceil((limit - (double)above_mass) / (double)w) : (double)count_in;
                nt = (uint32_t)fmin(fmax(more, 1.0), (double)count_in);
                if (kt == kk) nt = min(nt, kn);
            }
        }
    }
    const bool cut = kt != 0;

    // masses by segment, in index order
    const int per = (pieces + SEGS - 1) / SEGS, segs = (pieces + per - 1) / per;
    const double q = (double)s.q;
    for (int g = wave; g < segs; g += RW) {
        uint64_t m = 0;
        uint32_t ties = 0;
        for (int c = g * per; c < min((g + 1) * per, pieces); ++c) {
            float v[8];
            load8(x, mask, c * PIECE + lane * 8, n, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t key = key_of(v[e]);
                if (key > kt) {
                    const double w = W.real(v[e]);
                    m += w >= q ? W.fixed(w) : 0;
                }
                ties += cut && key == kt;
            }
        }
        m = wave_sum(m);
        ties = wave_sum(ties);
        if (lane == 0) {
            seg_mass[g] = m;
            seg_ties[g] = ties;
        }
    }
    __syncthreads();
    const double wt = cut ? W.real(of_key(kt)) : 0.0;
    const uint64_t wtie = wt >= q ? W.fixed(wt) : 0;
    const uint32_t mine = tid < segs ? seg_ties[tid] : 0;
    uint32_t all_ties;
    const uint32_t ties_ex = block_scan<uint32_t>(mine, scan32, all_ties);
    const uint32_t left = nt > ties_ex ? nt - ties_ex : 0;
    const uint64_t m = (tid < segs ? seg_mass[tid] : 0) + (uint64_t)min(mine, left) * wtie;
    uint64_t sum;
    const uint64_t m_ex = block_scan<uint64_t>(m, scan64, sum);
    const double target = (double)s.u * (double)sum;
    if ((double)(m_ex + m) > target && !((double)m_ex > target)) {   // one thread
        found_bin = (uint32_t)tid;
        found_mass = m_ex;
        found_count = ties_ex;
    }
    __syncthreads();
    if (wave != 0) return;

    // inside the segment
    uint64_t base = found_mass;
    uint32_t ties = found_count;
    const int g = (int)found_bin;
    for (int c = g * per; c < min((g + 1) * per, pieces); ++c) {
        float v[8];
        const int i = c * PIECE + lane * 8;
        load8(x, mask, i, n, v);
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) t += cut && key_of(v[e]) == kt;
        const uint32_t t_in = wave_scan(t, lane);
        uint32_t rank = ties + t_in - t;
        uint64_t w8[8], lane_mass = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t key = key_of(v[e]);
            w8[e] = 0;
            if (key > kt) {
                const double w = W.real(v[e]);
                w8[e] = w >= q ? W.fixed(w) : 0;
            } else if (cut && key == kt) {
                w8[e] = rank++ < nt ? wtie : 0;
            }
            lane_mass += w8[e];
        }
        const uint64_t in = wave_scan(lane_mass, lane);
        uint64_t upto = base + in - lane_mass;
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
        const uint64_t hits = __ballot(at >= 0);
        if (hits) {
            if (lane == __ffsll((unsigned long long)hits) - 1) answer(A, r, at, W.real(xa) * A.unit / (double)sum);
            return;
        }
        base += __shfl(in, 63);
        ties += __shfl(t_in, 63);
    }
}

static SampleArgs sample_args(const snk_sample_cfg_t *cfg, int64_t rows, int64_t n) {
    SNK_CHECK(cfg, SNK_ERR_INVALID, "sample: cfg is NULL");
    SNK_CHECK(cfg->struct_size == (int32_t)sizeof(snk_sample_cfg_t), SNK_ERR_INVALID,
              "snk_sample_cfg_t.struct_size = %d, the library's struct has %d bytes (binding out of date)",
              cfg->struct_size, (int)sizeof(snk_sample_cfg_t));
    SNK_CHECK(cfg->dtype == SNK_F32 || cfg->dtype == SNK_BF16 || cfg->dtype == SNK_F16, SNK_ERR_INVALID,
              "sample: unknown element type %d", cfg->dtype);
    SNK_CHECK(rows >= 0 && rows < (int64_t)1 << 31, SNK_ERR_INVALID, "sample: %lld rows", (long long)rows);
    SNK_CHECK(n >= 1 && n <= 1 << 24, SNK_ERR_INVALID, "sample: %lld logits a row, 1 to 2^24 are supported", (long long)n);
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
static void sample_launch_t(const SampleArgs &A, hipStream_t s) {
    const unsigned few = (unsigned)ceil_div(A.rows, 256);
    if (A.n <= 4)
        sample_few_kernel<T, 4><<<few, 256, 0, s>>>(A);
    else if (A.n <= 8)
        sample_few_kernel<T, 8><<<few, 256, 0, s>>>(A);
    else
        sample_row_kernel<T><<<(unsigned)A.rows, 1024, 0, s>>>(A);
    launch_check("sample kernel");
}

static void sample_launch(const SampleArgs &A, int32_t dtype, hipStream_t s) {
    if (A.rows == 0) return;
    if (dtype == SNK_F32)
        sample_launch_t<float>(A, s);
    else if (dtype == SNK_BF16)
        sample_launch_t<__bf16>(A, s);
    else
        sample_launch_t<_Float16>(A, s);
}

}  // namespace snk

using namespace snk;

extern "C" int snk_sample_workspace(int64_t rows, int64_t n, int64_t *bytes) {
    return guard([&] {
        SNK_CHECK(bytes && rows >= 0 && n >= 1, SNK_ERR_INVALID, "bad sample_workspace arguments");
        *bytes = 0;
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
        sample_launch(A, cfg->dtype, stream());
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
        sample_launch(A, SNK_F32, s);
    });
}
