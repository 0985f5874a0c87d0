// snk_optim.hip — AdamW over a list of tensors (include/snakehip.h), moments in 32 bits or in
// 8-bit codes with block scales.
//
// The step moves 28 B per fp32 element (p, m, v read and written, g read; 8-bit moments: 16 B, with
// 16-bit p and g 10 B) for ~20 operations, so HBM bounds it with 32-bit moments: every tensor is cut into chunks, a table holds each chunk's
// addresses, and one launch covers all tensors, whatever their number and sizes. A wave
// owns 256 consecutive elements (the 8-bit block), a lane four of them: 16-byte accesses, and the
// block's two scales are one wave reduction each.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstddef>
#include <cstring>
#include <memory>
#include <type_traits>
#include <vector>

#include "snk_optim.hpp"

namespace snk {

constexpr int BLK = 256;        // elements of a wave's block = the 8-bit states' block
constexpr int CH = 1024;        // elements of a workgroup's chunk
constexpr int NORM_WG = 1024;   // most workgroups (= partial sums) of the norm pass
// From this many bytes of parameters, gradients and moments on, a step reads and writes past the
// caches: nothing of them lives there until the next step, and what is written evicts nothing that is
// still to be read. 32-bit states: 159 us against 180 at 537 MB, 78 against 68 at 268 MB.
constexpr int64_t NT_FROM = 320ll << 20;
constexpr int64_t GRID = 1 << 23;   // chunks of one launch: the card's grids end at 2^32 threads
constexpr int FEW_PARTS = 256;  // partial sums that every workgroup of the step adds up itself

struct AdamTensor {
    void *p, *c;          // parameters, their rounded copy (or nullptr)
    const void *g;
};
struct alignas(16) AdamChunk {
    void *p, *c;          // at the chunk's first element
    int64_t place;        // in the state layout
    int64_t first;        // element of the tensor
    int32_t n, tensor;
    float wd;
    int32_t pad;
};
struct alignas(16) AdamCtl {
    int64_t t;            // the last step's number; if it was skipped, the next one takes it again
    double c1, c2;        // 1 - b^t
    int32_t skip;         // the last step's N was not finite
    float norm;           // the last step's N
    float ibc1, ibc2;     // 1 / (1 - b^t)
    float gmul;           // the factor of the gradients, where adamw_parts_kernel found it
    int32_t pad[3];
};
struct AdamHyper {
    double b1d, b2d;
    float b1, omb1, b2, omb2, eps, lr, gscale, max_norm;
    int32_t copy_dtype;
    uint64_t seed;
};

// An address that was itself loaded is generic to the compiler (flat accesses, waited for with LDS's):
// these go to global memory. N consecutive elements at an element-aligned address are one 16- or
// 8-byte access (unaligned global accesses are legal on gfx950), so views that start anywhere take
// the same path.
#define SNK_GLOBAL __attribute__((address_space(1)))
template <class T, int N>
struct Pack {
    typedef typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type Bits;
    typedef Bits Vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    Vec q;
    // NT: not kept in the caches (read or written once a step, and more of it than they hold)
    template <bool NT = false>
    __device__ __forceinline__ void load(const T *p) {
        q = NT ? __builtin_nontemporal_load((const SNK_GLOBAL Vec *)p) : *(const SNK_GLOBAL Vec *)p;
    }
    template <bool NT = false>
    __device__ __forceinline__ void store(T *p) const {
        if (NT)
            __builtin_nontemporal_store(q, (SNK_GLOBAL Vec *)p);
        else
            *(SNK_GLOBAL Vec *)p = q;
    }
    __device__ __forceinline__ float get(int k) const { return (float)__builtin_bit_cast(T, (Bits)q[k]); }
    __device__ __forceinline__ void set(int k, float x) { q[k] = __builtin_bit_cast(Bits, (T)x); }   // to nearest even
};
// four elements from place i of n, zeros behind the end; WHOLE: none lies there. Not converted yet: what
// is loaded next should not wait for this.
template <bool NT, class T, class I>
__device__ __forceinline__ Pack<T, 4> load4(const T *p, I i, I n, bool whole) {
    Pack<T, 4> q;
    if (whole) {
        q.template load<NT>(p + i);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) q.q[k] = i + k < n ? ((const SNK_GLOBAL typename Pack<T, 4>::Bits *)p)[i + k] : 0;
    }
    return q;
}
template <bool NT, class T, class I>
__device__ __forceinline__ void store4(T *p, I i, I n, bool whole, const float *x) {
    if (whole) {
        Pack<T, 4> q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q.set(k, x[k]);
        q.template store<NT>(p + i);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) ((SNK_GLOBAL T *)p)[i + k] = (T)x[k];
    }
}

// largest of 64 non-negative floats, which order as their bits do
__device__ __forceinline__ float wave_max_nonneg(float f) {
    uint32_t x = __float_as_uint(f);
    auto step = [&](auto ctrl) {   // 0 where a lane has no partner
        const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true);
        x = x > y ? x : y;
    };
    step(std::integral_constant<int, 0x111>{});   // row_shr 1, 2, 4, 8
    step(std::integral_constant<int, 0x112>{});
    step(std::integral_constant<int, 0x114>{});
    step(std::integral_constant<int, 0x118>{});
    step(std::integral_constant<int, 0x142>{});   // row_bcast 15, 31
    step(std::integral_constant<int, 0x143>{});
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)x, 63));
}

// the values the 8-bit codes stand for
__device__ __forceinline__ float m_value(float a, float scale) {   // a |a| / 127^2 (a |a| is exact)
    return a * fabsf(a) * (1.0f / 16129.0f) * scale;
}
__device__ __forceinline__ float v_level(float b) {   // (b / 255)^4
    const float r = b * (1.0f / 255.0f), r2 = r * r;
    return r2 * r2;
}
// x / d, correctly rounded, for many x and one d whose correctly rounded reciprocal is at hand: the
// quotient's residual is exact in an FMA, and one more rounds it (Markstein); d and x / d normal
__device__ __forceinline__ float quotient(float x, float d, float inv_d) {
    const float q = x * inv_d;
    return fmaf(fmaf(-q, d, x), inv_d, q);
}
// 1 / d, rounded correctly (but for a d whose significand is all ones): the hardware's (1 ulp) and a
// Newton step. d in the middle of fp32's range.
__device__ __forceinline__ float reciprocal(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.0f), r, r);
}
// a wave's largest value d >= 0 and the values brought there where they are not: far from an overflow of
// 1 / d and an underflow of what counts beside d
__device__ __forceinline__ void to_middle(float &d, float *x) {
    if (d >= 0x1p-100f && d <= 0x1p100f) return;
    asm volatile("");   // a branch that is hardly ever taken, not eight selects
    const float k = d < 1.0f ? 0x1p100f : 0x1p-100f;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= k;
    d = d > 0.0f ? d * k : 1.0f;
}

// what a step knows before it starts: its number and 1 / (1 - b^t)
struct AdamStep {
    int64_t t;
    double c1, c2;
    float ibc1, ibc2;
};
__host__ __device__ inline AdamStep next_step(int64_t t, double c1, double c2, const AdamHyper &H) {
    const double n1 = (1.0 - H.b1d) + H.b1d * c1, n2 = (1.0 - H.b2d) + H.b2d * c2;
    return AdamStep{t + 1, n1, n2, (float)(1.0 / n1), (float)(1.0 / n2)};
}

// the step's number and bias corrections, by one thread before the step's launch. In fp64: 1 - b^t
// loses digits in fp32 while t is small; 1 - b^t = (1 - b) + b (1 - b^(t-1)) needs no power.
__device__ __forceinline__ void begin_step(AdamCtl *ctl, const AdamHyper &H) {
    if (ctl->skip) return;   // that number has not been used
    const AdamStep n = next_step(ctl->t, ctl->c1, ctl->c2, H);
    ctl->t = n.t;
    ctl->c1 = n.c1;
    ctl->c2 = n.c2;
    ctl->ibc1 = n.ibc1;
    ctl->ibc2 = n.ibc2;
}
__global__ void adamw_begin_kernel(AdamCtl *__restrict__ ctl, AdamHyper H) { begin_step(ctl, H); }

// sum of a value over a workgroup of W waves, in one order, a wave's by lane moves; sh: W values
template <int CTRL, int ROWS>
__device__ __forceinline__ double plus_lane(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int W>
__device__ __forceinline__ double sum_group(double v, double *sh) {
    v = plus_lane<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8: within 16 lanes
    v = plus_lane<0x112, 0xf>(v);
    v = plus_lane<0x114, 0xf>(v);
    v = plus_lane<0x118, 0xf>(v);
    v = plus_lane<0x142, 0xa>(v);   // row_bcast 15, 31
    v = plus_lane<0x143, 0xc>(v);
    if ((threadIdx.x & 63) == 63) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = sh[0];
#pragma unroll
    for (int w = 1; w < W; ++w) sum += sh[w];
    return sum;
}

// N: partial sums of (s g)^2 in fp64 (fp32 squares overflow above 1.8e19 and lose the small ones).
// A wave a chunk, 16 elements a lane in 16-byte reads, the next chunk's record read ahead; bound by
// HBM's reads of g (133 M bf16: 73 us, 3.7 TB/s; 280 k fp32 2.7 us, the launch). The partials are added by the step itself or by adamw_parts_kernel: a count of
// arrivals costs more, 25 ns a workgroup (27 us for 1,079 of them). W waves a workgroup.
template <class GT, int W>
__global__ __launch_bounds__(64 * W) void adamw_norm_kernel(const AdamChunk *__restrict__ chunks, int64_t n_chunks,
                                                            const void *const *__restrict__ grads,
                                                            double *__restrict__ part, AdamCtl *__restrict__ ctl, AdamHyper H) {
    constexpr int V = 16 / sizeof(GT), N = CH / (64 * V);
    __shared__ double sh[W];
    const int lane = threadIdx.x & 63;
    const int64_t first = (int64_t)blockIdx.x * W + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t stride = (int64_t)gridDim.x * W;
    double sum = 0.0;
    const float gs = H.gscale;
    auto add = [&](float g) {
        const double d = (double)(g * gs);
        sum = fma(d, d, sum);
    };
    const GT *g = nullptr;
    int n = 0;
    if (first < n_chunks) {
        g = (const GT *)grads[first];
        n = chunks[first].n;
    }
    for (int64_t c = first; c < n_chunks; c += stride) {
        const int64_t next = c + stride < n_chunks ? c + stride : first;
        const GT *g_next = (const GT *)grads[next];
        const int n_next = chunks[next].n;
        if (n == CH) {
            Pack<GT, V> q[N];
#pragma unroll
            for (int j = 0; j < N; ++j) q[j].load(g + (j * 64 + lane) * V);
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) add(q[j].get(e));
        } else {   // whole vectors and the rest, all in flight at once
            Pack<GT, V> q[N];
            const int rest = n % V;
            GT x{};
#pragma unroll
            for (int j = 0; j < N; ++j) {
                q[j].q = 0;
                if ((j * 64 + lane + 1) * V <= n) q[j].load(g + (j * 64 + lane) * V);
            }
            if (lane < rest) x = ((const SNK_GLOBAL GT *)g)[n - rest + lane];
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) add(q[j].get(e));
            add((float)x);
        }
        g = g_next;
        n = n_next;
    }
    sum = sum_group<W>(sum, sh);
    if (threadIdx.x == 0) {
        part[blockIdx.x] = sum;
        if (blockIdx.x == 0) begin_step(ctl, H);
    }
}
// N and the factor of the gradients, s c; false where the step is to be skipped
__device__ __forceinline__ bool clip_factor(const AdamHyper &H, double sum, float &norm, float &gmul) {
    const double N = sqrt(sum);
    norm = (float)N;
    gmul = H.gscale;
    if (N > (double)H.max_norm) gmul = (float)((double)H.gscale * ((double)H.max_norm / N));
    return N < INFINITY;   // false for NaN too
}
// ... once for the whole step, where the partial sums are many
__global__ __launch_bounds__(256) void adamw_parts_kernel(const double *__restrict__ part, int n, AdamCtl *__restrict__ ctl,
                                                          AdamHyper H) {
    __shared__ double sh[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) sum += part[i];
    sum = sum_group<4>(sum, sh);
    if (threadIdx.x == 0) ctl->skip = clip_factor(H, sum, ctl->norm, ctl->gmul) ? 0 : 1;
}

struct AdamArgs {
    const AdamChunk *chunks;
    void *m, *v;
    float *ms, *vs;
    AdamCtl *ctl;
    const void *const *grads;   // each chunk's, as bound or as this call brought them
    const double *part;   // n_part partial sums of the norm (0: no norm, -1: ctl has its results)
    int n_part;
    bool counted;         // the host counts the steps: `step` holds, and ctl is to receive it
    AdamStep step;
    AdamHyper H;
};

__device__ __forceinline__ AdamStep this_step(const AdamArgs &A) {
    if (!A.counted) return AdamStep{A.ctl->t, A.ctl->c1, A.ctl->c2, A.ctl->ibc1, A.ctl->ibc2};
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        A.ctl->t = A.step.t;
        A.ctl->c1 = A.step.c1;
        A.ctl->c2 = A.step.c2;
    }
    return A.step;
}

// the factor of the gradients, s c; false where the step is skipped. Workgroup 0 records N.
__device__ __forceinline__ double own_part(const AdamArgs &A) {   // before what takes longer to arrive
    return (int)threadIdx.x < A.n_part ? A.part[threadIdx.x] : 0.0;
}
__device__ __forceinline__ bool grad_factor(const AdamArgs &A, double part, double *sh, float &gmul) {
    gmul = A.H.gscale;
    if (A.n_part == 0) return true;
    if (A.n_part < 0) {
        gmul = A.ctl->gmul;
        return A.ctl->skip == 0;
    }
    const double sum = sum_group<4>(part, sh);
    float norm;
    const bool fine = clip_factor(A.H, sum, norm, gmul);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        A.ctl->norm = norm;
        A.ctl->skip = fine ? 0 : 1;
    }
    return fine;
}

// one element: new moments in m, v; the new parameter is returned. EXACT: the step's root and quotient
// correctly rounded (HBM hides them with 32-bit moments), or within an ulp each by the hardware's own,
// which take a subnormal v for 0: nothing beside an eps of 1e-12 and more
template <bool EXACT>
__device__ __forceinline__ float adamw_one(const AdamHyper &H, float gmul, float ibc1, float ibc2, float wd, float p,
                                           float g, float &m, float &v) {
    g *= gmul;
    m = H.b1 * m + H.omb1 * g;
    v = H.b2 * v + H.omb2 * (g * g);
    const float den = (EXACT ? __builtin_sqrtf(v * ibc2) : __builtin_amdgcn_sqrtf(v * ibc2)) + H.eps;
    const float step = EXACT ? (m * ibc1) / den : (m * ibc1) * __builtin_amdgcn_rcpf(den);
    return p - H.lr * (step + wd * p);
}

template <class PT, bool NT>
__device__ __forceinline__ void store_params(const AdamChunk &T, int copy_dtype, int i, bool whole, const float *p) {
    store4<NT>((PT *)T.p, i, T.n, whole, p);
    if (T.c) {
        if (copy_dtype == SNK_BF16)
            store4<NT>((__bf16 *)T.c, i, T.n, whole, p);
        else
            store4<NT>((_Float16 *)T.c, i, T.n, whole, p);
    }
}

// A workgroup a chunk, its p, g, m and v loaded before any is used. Waves behind the chunk's end read its
// last 256 places too, so that no load waits for a test, and leave before the first store. 133 M fp32
// parameters, bf16 gradients: 545 us, 3.47 GB at 6.4 TB/s (a copy of 4 GiB: 4.7); through the caches 650.
template <class PT, class GT, bool NT>
__global__ __launch_bounds__(256) void adamw32_kernel(AdamArgs A) {
    __shared__ double sh[4];
    const AdamChunk T = A.chunks[blockIdx.x];
    const GT *const g = (const GT *)A.grads[blockIdx.x];
    const AdamStep now = this_step(A);
    const float ibc1 = now.ibc1, ibc2 = now.ibc2;
    const int lane = threadIdx.x & 63, mine = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int last = (T.n - 1) / BLK, wave = mine < last ? mine : last;
    const int i = wave * BLK + lane * 4;
    const bool whole = (wave + 1) * BLK <= T.n;
    float *ms = (float *)A.m + T.place, *vs = (float *)A.v + T.place;
    const double part = own_part(A);
    Pack<float, 4> mq, vq;
    mq.template load<NT>(ms + i);   // padded: always whole
    vq.template load<NT>(vs + i);
    const Pack<PT, 4> pq = load4<NT>((const PT *)T.p, i, T.n, whole);
    const Pack<GT, 4> gq = load4<NT>(g, i, T.n, whole);
    float gmul;
    if (!grad_factor(A, part, sh, gmul) || mine > last) return;
    float p[4], m[4], v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        m[e] = mq.get(e);
        v[e] = vq.get(e);
        p[e] = adamw_one<true>(A.H, gmul, ibc1, ibc2, T.wd, pq.get(e), gq.get(e), m[e], v[e]);
        mq.set(e, m[e]);
        vq.set(e, v[e]);
    }
    mq.template store<NT>(ms + i);
    vq.template store<NT>(vs + i);
    store_params<PT, NT>(T, A.H.copy_dtype, i, whole, p);
}

// The same with 8-bit moments, a wave a block of them. 133 M bf16 parameters and gradients: 297 us,
// 1.33 GB at 4.5 TB/s: HBM and, next to it, the 326 vector instructions of a wave (four elements a lane,
// half of them for the codes: 280 us if they issued without a pause). Divides and roots by the compiler's
// sequences took 580 us, loads that wait for one another 408.
template <class PT, class GT, bool NT>
__global__ __launch_bounds__(256) void adamw8_kernel(AdamArgs A) {
    __shared__ double sh[4];
    __shared__ float level[256];   // v's: 12 multiplications an element that one read and one pair of reads do
    const AdamChunk T = A.chunks[blockIdx.x];
    const GT *const g = (const GT *)A.grads[blockIdx.x];
    const AdamStep now = this_step(A);
    const float ibc1 = now.ibc1, ibc2 = now.ibc2;
    const int lane = threadIdx.x & 63, mine = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int last = (T.n - 1) / BLK, wave = mine < last ? mine : last;
    const int i = wave * BLK + lane * 4;
    const bool whole = (wave + 1) * BLK <= T.n;
    const uint64_t key = splitmix64(A.H.seed ^ ((uint64_t)now.t * 0xD1B54A32D192ED03ULL));   // rng_hash's first half
    const int64_t block = T.place / BLK + wave;
    SNK_GLOBAL uint32_t *mcs = (SNK_GLOBAL uint32_t *)A.m + block * 64, *vcs = (SNK_GLOBAL uint32_t *)A.v + block * 64;
    const double part = own_part(A);
    uint32_t mc, vc;
    if (NT) {
        mc = __builtin_nontemporal_load(mcs + lane);
        vc = __builtin_nontemporal_load(vcs + lane);
    } else {
        mc = mcs[lane];
        vc = vcs[lane];
    }
    const Pack<PT, 4> pq = load4<NT>((const PT *)T.p, i, T.n, whole);
    const Pack<GT, 4> gq = load4<NT>(g, i, T.n, whole);
    const float ms0 = A.ms[block], vs0 = A.vs[block];
    level[threadIdx.x] = v_level((float)threadIdx.x);
    const uint64_t h = splitmix64(key ^ (uint64_t)(block * 64 + lane));
    float gmul;
    const bool go = grad_factor(A, part, sh, gmul);
    __syncthreads();
    if (!go || mine > last) return;
    float p[4], m[4], v[4], mmax = 0.0f, vmax = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {   // places behind the tensor's end hold zeros and read g = 0
        m[e] = m_value((float)(int8_t)(mc >> (8 * e)), ms0);
        v[e] = level[(vc >> (8 * e)) & 255u] * vs0;
        p[e] = adamw_one<false>(A.H, gmul, ibc1, ibc2, T.wd, pq.get(e), gq.get(e), m[e], v[e]);
        mmax = fmaxf(mmax, fabsf(m[e]));
        vmax = fmaxf(vmax, v[e]);
    }
    store_params<PT, NT>(T, A.H.copy_dtype, i, whole, p);
    mmax = wave_max_nonneg(mmax);
    vmax = wave_max_nonneg(vmax);
    if (fmaxf(mmax, vmax) == INFINITY) {   // the whole wave, hardly ever: no scale is infinite
        mmax = vmax = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (fabsf(m[e]) == INFINITY) m[e] = v[e] = 0.0f;   // with it the parameter was lost, and no other is
            if (v[e] == INFINITY) v[e] = FLT_MAX;              // of a finite gradient: its next steps stay small
            mmax = fmaxf(mmax, fabsf(m[e]));
            vmax = fmaxf(vmax, v[e]);
        }
        mmax = wave_max_nonneg(mmax);
        vmax = wave_max_nonneg(vmax);
    }
    // The codes as correctly rounded quotients and roots give them (the same arithmetic anywhere gives
    // the same codes): by one reciprocal a wave, of a scale in the middle of fp32's range.
    float least[4], dm = mmax, dv = vmax;
#pragma unroll
    for (int e = 0; e < 4; ++e) least[e] = __builtin_amdgcn_fmed3f(ceilf(v[e]), 0.0f, 1.0f);
    to_middle(dm, m);
    to_middle(dv, v);
    const float im = reciprocal(dm), iv = reciprocal(dv);
    uint32_t mo = 0, vo = 0;
    float a[4], far = 0.0f, all = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x = 127.0f * __builtin_amdgcn_sqrtf(fabsf(m[e]) * im);   // within 127 2^-22 of the true one
        a[e] = rintf(x);
        far = fmaxf(far, fabsf(x - a[e]));
        all += x - a[e];   // NaN where an x is
    }
    // 1 wave in 20: what is next to a half (and a NaN, whose code is 0), again in full
    if (__builtin_amdgcn_ballot_w64(!(fmaf(0.0f, all, far) < 0.4999f)))
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = rintf(127.0f * __builtin_sqrtf(fmaxf(fabsf(m[e]) / dm, 0.0f)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        mo = __builtin_amdgcn_cvt_pk_u8_f32(copysignf(a[e], m[e]) + 128.0f, e, mo);
        // next to a level either floor leads to that level, so the hardware's roots (1 ulp) do here. What
        // is above 0 never becomes 0 (m / eps would follow): its lower level is at least the first.
        const float part = quotient(v[e], dv, iv);
        const float low = __builtin_amdgcn_fmed3f(floorf(255.0f * __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(part))), least[e], 254.0f);
        const int l = (int)low;
        const float lo = level[l], hi = level[l + 1];
        const float r = (float)((uint32_t)(h >> (16 * e)) & 0xFFFFu) * 0x1p-16f;
        vo = __builtin_amdgcn_cvt_pk_u8_f32(r * (hi - lo) < part - lo ? low + 1.0f : low, e, vo);
    }
    mo ^= 0x80808080u;   // a + 128 as a signed byte
    if (NT) {
        __builtin_nontemporal_store(mo, mcs + lane);
        __builtin_nontemporal_store(vo, vcs + lane);
    } else {
        mcs[lane] = mo;
        vcs[lane] = vo;
    }
    if (lane == 0) {
        A.ms[block] = mmax;
        A.vs[block] = vmax;
    }
}

// The moments' values, a lane four places. 133 M of 8 bits to bf16: 150 us, 0.80 GB at 5.3 TB/s.
template <class OT, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_moments_kernel(AdamArgs A, int64_t total, OT *__restrict__ mo,
                                                            OT *__restrict__ vo) {
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < total; i += (int64_t)gridDim.x * 1024) {
        const bool whole = i + 4 <= total;
        float m[4], v[4];
        if (EIGHT) {
            const uint32_t mc = *(const uint32_t *)((const uint8_t *)A.m + i);
            const uint32_t vc = *(const uint32_t *)((const uint8_t *)A.v + i);
            const float ms = A.ms[i / BLK], vs = A.vs[i / BLK];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = m_value((float)(int8_t)(mc >> (8 * e)), ms);
                v[e] = v_level((float)((vc >> (8 * e)) & 255u)) * vs;
            }
        } else {
            const Pack<float, 4> mq = load4<false>((const float *)A.m, i, total, whole);
            const Pack<float, 4> vq = load4<false>((const float *)A.v, i, total, whole);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = mq.get(e);
                v[e] = vq.get(e);
            }
        }
        if (mo) store4<false>(mo, i, total, whole, m);
        if (vo) store4<false>(vo, i, total, whole, v);
    }
}

// tensor addresses into the device table, by value: safe inside a capture, where a host array
// would be read again at every replay
constexpr int BIND_N = 128, GIVEN_N = 384;   // 3 KB of arguments each
struct BindArgs {
    void *p[BIND_N], *c[BIND_N];
    const void *g[BIND_N];
};
__global__ void adamw_bind_kernel(AdamTensor *__restrict__ tab, BindArgs b, int n) {
    const int i = threadIdx.x;
    if (i < n) {
        tab[i].p = b.p[i];
        tab[i].g = b.g[i];
        tab[i].c = b.c[i];
    }
}
struct GivenArgs {
    const void *g[GIVEN_N];
};
// The gradients' addresses of the chunks first..n - 1, which are those of the tensors at..at + GIVEN_N - 1:
// 5 us for 130,000 chunks, 2 to 2.6 for few. An address a chunk, not a tensor: where every workgroup looked its
// tensor's up behind the chunk's record, a step of 133 M bf16 parameters with 8-bit moments, and the moments
// read out, took 513 us instead of 498.
__global__ __launch_bounds__(256) void adamw_given_kernel(const AdamChunk *__restrict__ chunks, const void **__restrict__ grads,
                                                          GivenArgs b, int at, int64_t first, int64_t n, int gsize) {
    const int64_t k = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (k < n) grads[k] = (const uint8_t *)b.g[chunks[k].tensor - at] + chunks[k].first * gsize;
}
__global__ __launch_bounds__(256) void adamw_chunks_kernel(const AdamTensor *__restrict__ tab, AdamChunk *__restrict__ chunks,
                                                           const void **__restrict__ grads, int64_t n, int psize, int gsize) {
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (k >= n) return;
    AdamChunk &c = chunks[k];
    const AdamTensor t = tab[c.tensor];
    c.p = (uint8_t *)t.p + c.first * psize;
    grads[k] = (const uint8_t *)t.g + c.first * gsize;
    c.c = t.c ? (uint8_t *)t.c + c.first * 2 : nullptr;
}
__global__ void adamw_fill_kernel(uint32_t *__restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = 0;
}

struct AdamSpan {   // of addresses
    uintptr_t lo, hi;
    bool written;
};

}  // namespace snk

using namespace snk;

struct snk_adamw_s {
    snk_adamw_cfg_t cfg{};
    int device = 0;
    bool owned = false, bound = false;
    bool grads_bound = false;
    bool captured = false;   // a step was captured: only the device knows the count
    AdamStep now{};          // the count until then, without a norm
    std::vector<int64_t> size, start, first_chunk;
    int64_t total = 0, n_chunks = 0;
    std::vector<AdamSpan> written;   // the bound parameters and copies, by address
    DevBuf<AdamTensor> tab;
    DevBuf<const void *> bound_grads, given_grads;   // each chunk's: as bound, of the last step that brought its own
    DevBuf<AdamChunk> chunks;
    DevBuf<uint8_t> m, v;
    DevBuf<float> ms, vs;
    DevBuf<double> part;
    DevBuf<AdamCtl> ctl;
    int64_t state_bytes() const { return total * (cfg.state_bits / 8); }
    AdamArgs args() const {
        AdamArgs a{};
        a.chunks = chunks.p;
        a.m = m.p;
        a.v = v.p;
        a.ms = ms.p;
        a.vs = vs.p;
        a.ctl = ctl.p;
        a.part = part.p;
        return a;
    }
};

static int dtype_size(int32_t d) { return d == SNK_F32 ? 4 : 2; }   // bytes
static bool dtype_ok(int32_t d) { return d == SNK_F32 || d == SNK_BF16 || d == SNK_F16; }

static void check_device(snk_adamw h) {
    int dev = 0;
    SNK_HIP(hipGetDevice(&dev));
    SNK_CHECK(dev == h->device, SNK_ERR_STATE, "the AdamW handle lives on device %d, the current device is %d", h->device,
              dev);
}

namespace snk {

// what a replay would not do again, what would leave addresses that no replay has brought yet, and what
// waits for the stream, which would end the capture
void adamw_not_captured(hipStream_t s, const char *what) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    SNK_HIP(hipStreamIsCapturing(s, &st));
    SNK_CHECK(st == hipStreamCaptureStatusNone, SNK_ERR_STATE, "AdamW: %s while the stream is being captured", what);
}

void adamw_reset(snk_adamw h, hipStream_t s) {
    auto zero = [&](void *p, int64_t bytes) {   // a kernel, not hipMemsetAsync: callers may capture
        if (bytes == 0) return;
        adamw_fill_kernel<<<(unsigned)std::min<int64_t>(ceil_div(bytes / 4, 256), 2048), 256, 0, s>>>((uint32_t *)p, bytes / 4);
        launch_check("adamw_fill_kernel");
    };
    zero(h->m, h->state_bytes());
    zero(h->v, h->state_bytes());
    if (h->cfg.state_bits == 8) {
        zero(h->ms, h->total / BLK * 4);
        zero(h->vs, h->total / BLK * 4);
    }
    zero(h->ctl, sizeof(AdamCtl));
    h->now = AdamStep{};
}

snk_adamw adamw_create(int32_t n, const int64_t *sizes, const float *wd, const snk_adamw_cfg_t *cfg) {
    SNK_CHECK(n > 0 && sizes && wd && cfg, SNK_ERR_INVALID, "bad adamw_create arguments");
    SNK_CHECK(cfg->struct_size == (int32_t)sizeof(snk_adamw_cfg_t), SNK_ERR_INVALID,
              "snk_adamw_cfg_t.struct_size = %d, the library's struct has %d bytes (binding out of date)",
              cfg->struct_size, (int)sizeof(snk_adamw_cfg_t));
    SNK_CHECK(dtype_ok(cfg->param_dtype) && dtype_ok(cfg->grad_dtype), SNK_ERR_INVALID, "AdamW: unknown element type");
    SNK_CHECK(cfg->copy_dtype == -1 || cfg->copy_dtype == SNK_BF16 || cfg->copy_dtype == SNK_F16, SNK_ERR_INVALID,
              "AdamW: copy_dtype %d is not -1, bf16 or fp16", cfg->copy_dtype);
    SNK_CHECK(cfg->state_bits == 32 || cfg->state_bits == 8, SNK_ERR_INVALID, "AdamW: state_bits %d is not 32 or 8",
              cfg->state_bits);
    SNK_CHECK(cfg->beta1 >= 0 && cfg->beta1 < 1 && cfg->beta2 >= 0 && cfg->beta2 < 1, SNK_ERR_INVALID,
              "AdamW: betas (%g, %g) outside [0, 1)", cfg->beta1, cfg->beta2);
    const double least = cfg->state_bits == 8 ? 1e-12 : 1e-30;
    SNK_CHECK(cfg->eps >= least && cfg->eps <= 1e30, SNK_ERR_INVALID, "AdamW: eps %g outside [%g, 1e30]", cfg->eps, least);
    SNK_CHECK(cfg->max_grad_norm >= 0, SNK_ERR_INVALID, "AdamW: max_grad_norm %g is negative", cfg->max_grad_norm);
    SNK_CHECK(cfg->reserved == 0, SNK_ERR_INVALID, "AdamW: reserved must be 0");
    hipStream_t s = stream();
    adamw_not_captured(s, "a handle is made");
    auto h = std::make_unique<snk_adamw_s>();
    h->cfg = *cfg;
    SNK_HIP(hipGetDevice(&h->device));
    for (int i = 0; i < n; ++i) {
        SNK_CHECK(sizes[i] >= 0 && sizes[i] < (int64_t)1 << 40 && h->total < (int64_t)1 << 40, SNK_ERR_INVALID,
                  "AdamW: tensor %d has %lld elements", i, (long long)sizes[i]);
        SNK_CHECK(wd[i] >= 0 && wd[i] < INFINITY, SNK_ERR_INVALID, "AdamW: weight decay %g of tensor %d", wd[i], i);
        h->size.push_back(sizes[i]);
        h->start.push_back(h->total);
        h->total += (sizes[i] + BLK - 1) / BLK * BLK;
        h->first_chunk.push_back(h->n_chunks);
        h->n_chunks += (sizes[i] + CH - 1) / CH;
    }
    h->first_chunk.push_back(h->n_chunks);
    SNK_CHECK(h->n_chunks < (int64_t)1 << 31, SNK_ERR_INVALID, "AdamW: too many elements for one handle");
    std::vector<AdamChunk> chunks;
    for (int i = 0; i < n; ++i)
        for (int64_t at = 0; at < sizes[i]; at += CH)
            chunks.push_back(AdamChunk{nullptr, nullptr, h->start[i] + at, at, (int32_t)std::min<int64_t>(CH, sizes[i] - at),
                                       i, wd[i], 0});
    h->tab = DevBuf<AdamTensor>(n);
    h->chunks = DevBuf<AdamChunk>(chunks.size());
    h->bound_grads = DevBuf<const void *>(chunks.size());
    h->given_grads = DevBuf<const void *>(chunks.size());
    h->m = DevBuf<uint8_t>(h->state_bytes());
    h->v = DevBuf<uint8_t>(h->state_bytes());
    if (cfg->state_bits == 8) {
        h->ms = DevBuf<float>(h->total / BLK);
        h->vs = DevBuf<float>(h->total / BLK);
    }
    h->part = DevBuf<double>(NORM_WG);
    h->ctl = DevBuf<AdamCtl>(1);
    if (!chunks.empty())
        SNK_HIP(hipMemcpyAsync(h->chunks, chunks.data(), chunks.size() * sizeof(AdamChunk), hipMemcpyHostToDevice, s));
    adamw_reset(h.get(), s);
    SNK_HIP(hipStreamSynchronize(s));
    return h.release();
}

void adamw_free(snk_adamw h) { delete h; }
void adamw_set_owned(snk_adamw h) { h->owned = true; }

static AdamSpan span_of(const void *p, int64_t size, int32_t dtype, bool written, const char *what, int i) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    SNK_CHECK(a && a % dtype_size(dtype) == 0, SNK_ERR_INVALID, "AdamW: %s %d is NULL or not element-aligned", what, i);
    return AdamSpan{a, a + (uintptr_t)size * dtype_size(dtype), written};
}

void adamw_bind(snk_adamw h, void *const *params, const void *const *grads, void *const *copies, hipStream_t s) {
    const int n = (int)h->size.size();
    SNK_CHECK(params, SNK_ERR_INVALID, "adamw_bind: NULL argument");
    adamw_not_captured(s, "tensors are bound");
    SNK_CHECK(grads || !h->grads_bound, SNK_ERR_STATE,
              "adamw_bind: this handle's gradients are bound, and captured steps may read them: bind others");
    SNK_CHECK((copies != nullptr) == (h->cfg.copy_dtype >= 0), SNK_ERR_INVALID,
              "adamw_bind: copies go with a copy_dtype, and only with one");
    std::vector<AdamSpan> spans;
    auto add = [&](const void *p, int i, int32_t dtype, bool written, const char *what) {
        if (h->size[i] == 0) return;
        spans.push_back(span_of(p, h->size[i], dtype, written, what, i));
    };
    for (int i = 0; i < n; ++i) {
        add(params[i], i, h->cfg.param_dtype, true, "parameter");
        if (grads) add(grads[i], i, h->cfg.grad_dtype, false, "gradient");
        if (copies) add(copies[i], i, h->cfg.copy_dtype, true, "copy");
    }
    // a tensor that is written must not overlap any other: the chunks run in no order. Swept by
    // address with the furthest end seen of all spans and of the written ones
    std::sort(spans.begin(), spans.end(), [](const AdamSpan &a, const AdamSpan &b) { return a.lo < b.lo; });
    uintptr_t end = 0, end_written = 0;
    for (const AdamSpan &x : spans) {
        SNK_CHECK(x.lo >= end_written && !(x.written && x.lo < end), SNK_ERR_INVALID,
                  "adamw_bind: a parameter or copy overlaps another tensor");
        end = std::max(end, x.hi);
        if (x.written) end_written = std::max(end_written, x.hi);
    }
    for (int at = 0; at < n; at += BIND_N) {
        BindArgs b{};
        const int k = std::min(BIND_N, n - at);
        for (int i = 0; i < k; ++i) {
            b.p[i] = params[at + i];
            b.g[i] = grads ? grads[at + i] : nullptr;
            b.c[i] = copies ? copies[at + i] : nullptr;
        }
        adamw_bind_kernel<<<1, BIND_N, 0, s>>>(h->tab + at, b, k);
        launch_check("adamw_bind_kernel");
    }
    if (h->n_chunks > 0) {
        adamw_chunks_kernel<<<(unsigned)ceil_div(h->n_chunks, 256), 256, 0, s>>>(
            h->tab, h->chunks, h->bound_grads, h->n_chunks, dtype_size(h->cfg.param_dtype), dtype_size(h->cfg.grad_dtype));
        launch_check("adamw_chunks_kernel");
    }
    spans.erase(std::remove_if(spans.begin(), spans.end(), [](const AdamSpan &x) { return !x.written; }), spans.end());
    h->written.swap(spans);
    h->bound = true;
    h->grads_bound = grads != nullptr;
}

template <class F>
static void with_type(int32_t d, F &&f) {
    if (d == SNK_F32)
        f(float{});
    else if (d == SNK_BF16)
        f(__bf16{});
    else
        f(_Float16{});
}

// this step's own gradients to their chunks: one launch for up to GIVEN_N tensors
static void give_grads(snk_adamw h, int32_t dtype, const void *const *grads, hipStream_t s) {
    const int n = (int)h->size.size();
    for (int i = 0; i < n; ++i) {
        if (h->size[i] == 0) continue;
        const AdamSpan x = span_of(grads[i], h->size[i], dtype, false, "gradient", i);
        // of the written spans, none of which overlap, the first that ends behind x's start
        const auto w = std::upper_bound(h->written.begin(), h->written.end(), x.lo,
                                        [](uintptr_t a, const AdamSpan &b) { return a < b.hi; });
        SNK_CHECK(w == h->written.end() || w->lo >= x.hi, SNK_ERR_INVALID, "AdamW: gradient %d overlaps a parameter or copy", i);
    }
    for (int at = 0; at < n; at += GIVEN_N) {
        GivenArgs b{};
        const int k = std::min(GIVEN_N, n - at);
        std::copy(grads + at, grads + at + k, b.g);
        const int64_t first = h->first_chunk[at], end = h->first_chunk[at + k];
        if (first == end) continue;
        adamw_given_kernel<<<(unsigned)ceil_div(end - first, 256), 256, 0, s>>>(h->chunks, h->given_grads, b, at, first, end,
                                                                             dtype_size(dtype));
        launch_check("adamw_given_kernel");
    }
}

void adamw_step(snk_adamw h, float lr, float grad_scale, hipStream_t s, int32_t grad_dtype, const void *const *grads) {
    SNK_CHECK(h->bound, SNK_ERR_STATE, "AdamW: no tensors are bound");
    SNK_CHECK(grads || h->grads_bound, SNK_ERR_STATE, "AdamW: no gradients are bound or given");
    SNK_CHECK(lr >= 0 && lr < INFINITY && std::isfinite(grad_scale), SNK_ERR_INVALID, "AdamW: lr %g, grad_scale %g", lr,
              grad_scale);
    const snk_adamw_cfg_t &c = h->cfg;
    AdamArgs A = h->args();
    if (grads) {
        SNK_CHECK(dtype_ok(grad_dtype), SNK_ERR_INVALID, "AdamW: unknown element type");
        give_grads(h, grad_dtype, grads, s);
        A.grads = h->given_grads;
    } else {
        grad_dtype = c.grad_dtype;
        A.grads = h->bound_grads;
    }
    AdamHyper &H = A.H;
    H.b1d = c.beta1;
    H.b2d = c.beta2;
    H.b1 = (float)c.beta1;
    H.omb1 = (float)(1.0 - c.beta1);
    H.b2 = (float)c.beta2;
    H.omb2 = (float)(1.0 - c.beta2);
    H.eps = (float)c.eps;
    H.lr = lr;
    H.gscale = grad_scale;
    H.max_norm = c.max_grad_norm;
    H.copy_dtype = c.copy_dtype;
    H.seed = c.seed;
    if (c.max_grad_norm > 0 && h->n_chunks > 0) {
        // a chunk a wave as long as the step can add the partial sums itself: workgroups of four waves,
        // or of eight (1.1 M elements: 14.6 us a step against 15.7; 490 k: 10.0 against 9.8)
        const bool eight = h->n_chunks > 4 * FEW_PARTS;
        const int64_t groups = eight ? (h->n_chunks + 7) / 8 : (h->n_chunks + 3) / 4;
        int parts = (int)std::min<int64_t>(groups, groups <= 2 * FEW_PARTS ? FEW_PARTS : NORM_WG);
        with_type(grad_dtype, [&](auto g) {
            using GT = decltype(g);
            if (eight)
                adamw_norm_kernel<GT, 8><<<(unsigned)parts, 512, 0, s>>>(h->chunks, h->n_chunks, A.grads, h->part, h->ctl, H);
            else
                adamw_norm_kernel<GT, 4><<<(unsigned)parts, 256, 0, s>>>(h->chunks, h->n_chunks, A.grads, h->part, h->ctl, H);
        });
        launch_check("adamw_norm_kernel");
        if (parts > FEW_PARTS) {
            adamw_parts_kernel<<<1, 256, 0, s>>>(h->part, parts, h->ctl, H);
            launch_check("adamw_parts_kernel");
            parts = -1;
        }
        A.n_part = parts;
    } else {
        // no norm, so no step is skipped, and the host can count them itself (a launch fewer) as long
        // as none was captured: replays would not pass by here
        if (!h->captured) {
            hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
            SNK_HIP(hipStreamIsCapturing(s, &st));
            h->captured = st != hipStreamCaptureStatusNone;
        }
        if (h->captured || h->n_chunks == 0) {
            h->captured = true;
            adamw_begin_kernel<<<1, 1, 0, s>>>(h->ctl, H);
            launch_check("adamw_begin_kernel");
        } else {
            A.counted = true;
            A.step = h->now = next_step(h->now.t, h->now.c1, h->now.c2, H);
        }
    }
    if (h->n_chunks == 0) return;
    const bool nt = h->total * (dtype_size(c.param_dtype) + dtype_size(grad_dtype) + c.state_bits / 4) >= NT_FROM;
    for (int64_t at = 0; at < h->n_chunks; at += GRID, A.chunks += GRID, A.grads += GRID) {
        with_type(c.param_dtype, [&](auto p) {
            with_type(grad_dtype, [&](auto g) {
                using PT = decltype(p);
                using GT = decltype(g);
                const unsigned grid = (unsigned)std::min(GRID, h->n_chunks - at);
                if (c.state_bits == 8 && nt)
                    adamw8_kernel<PT, GT, true><<<grid, 256, 0, s>>>(A);
                else if (c.state_bits == 8)
                    adamw8_kernel<PT, GT, false><<<grid, 256, 0, s>>>(A);
                else if (nt)
                    adamw32_kernel<PT, GT, true><<<grid, 256, 0, s>>>(A);
                else
                    adamw32_kernel<PT, GT, false><<<grid, 256, 0, s>>>(A);
            });
        });
        launch_check("adamw_kernel");
    }
}

}  // namespace snk

extern "C" int snk_adamw_create(snk_adamw *out, int32_t n, const int64_t *sizes, const float *wd,
                                const snk_adamw_cfg_t *cfg) {
    return guard([&] {
        SNK_CHECK(out, SNK_ERR_INVALID, "out is NULL");
        *out = adamw_create(n, sizes, wd, cfg);
    });
}

extern "C" int snk_adamw_destroy(snk_adamw h) {
    return guard([&] {
        if (!h) return;
        SNK_CHECK(!h->owned, SNK_ERR_STATE, "the AdamW handle belongs to a model (snk_dqn_use_adamw)");
        (void)hipDeviceSynchronize();   // its steps may be in flight on any stream
        adamw_free(h);
    });
}

extern "C" int snk_adamw_bind(snk_adamw h, void *const *params, const void *const *grads, void *const *copies) {
    return guard([&] {
        SNK_CHECK(h, SNK_ERR_INVALID, "NULL argument");
        SNK_CHECK(!h->owned, SNK_ERR_STATE, "the AdamW handle belongs to a model (snk_dqn_use_adamw)");
        check_device(h);
        adamw_bind(h, params, grads, copies, stream());
    });
}

extern "C" int snk_adamw_step(snk_adamw h, float lr, float grad_scale) {
    return guard([&] {
        SNK_CHECK(h, SNK_ERR_INVALID, "NULL argument");
        SNK_CHECK(!h->owned, SNK_ERR_STATE, "the AdamW handle belongs to a model: snk_dqn_apply_grad steps it");
        check_device(h);
        adamw_step(h, lr, grad_scale, stream());
    });
}

extern "C" int snk_adamw_step_grads(snk_adamw h, int32_t grad_dtype, const void *const *grads, float lr, float grad_scale) {
    return guard([&] {
        SNK_CHECK(h && grads, SNK_ERR_INVALID, "NULL argument");
        SNK_CHECK(!h->owned, SNK_ERR_STATE, "the AdamW handle belongs to a model: snk_dqn_apply_grad steps it");
        check_device(h);
        adamw_step(h, lr, grad_scale, stream(), grad_dtype, grads);
    });
}

extern "C" int snk_adamw_layout(snk_adamw h, int64_t *total, int64_t *starts) {
    return guard([&] {
        SNK_CHECK(h && total, SNK_ERR_INVALID, "NULL argument");
        *total = h->total;
        if (starts) std::copy(h->start.begin(), h->start.end(), starts);
    });
}

extern "C" int snk_adamw_state_ptr(snk_adamw h, int32_t which, void **dev_out, int64_t *bytes_out) {
    return guard([&] {
        SNK_CHECK(h && dev_out && bytes_out, SNK_ERR_INVALID, "NULL argument");
        const bool scales = which == SNK_ADAMW_M_SCALE || which == SNK_ADAMW_V_SCALE;
        SNK_CHECK(which >= SNK_ADAMW_M && which <= SNK_ADAMW_NORM && (!scales || h->cfg.state_bits == 8), SNK_ERR_INVALID,
                  "AdamW: no state %d", which);
        void *const p[] = {h->m.p, h->v.p, h->ms.p, h->vs.p, &h->ctl.p->norm};
        *dev_out = p[which];
        *bytes_out = which == SNK_ADAMW_NORM ? 4 : scales ? h->total / BLK * 4 : h->state_bytes();
    });
}

extern "C" int snk_adamw_moments(snk_adamw h, int32_t dtype, void *m_dev, void *v_dev) {
    return guard([&] {
        SNK_CHECK(h && dtype_ok(dtype), SNK_ERR_INVALID, "bad adamw_moments arguments");
        check_device(h);
        if (h->total == 0 || (!m_dev && !v_dev)) return;
        const uintptr_t a = reinterpret_cast<uintptr_t>(m_dev), b = reinterpret_cast<uintptr_t>(v_dev);
        const uintptr_t bytes = (uintptr_t)h->total * dtype_size(dtype);
        SNK_CHECK(a % dtype_size(dtype) == 0 && b % dtype_size(dtype) == 0, SNK_ERR_INVALID,
                  "adamw_moments: an array is not element-aligned");
        SNK_CHECK(!a || !b || a + bytes <= b || b + bytes <= a, SNK_ERR_INVALID,
                  "adamw_moments: both moments into one array, or arrays that overlap");
        const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(h->total, 1024), 4096);
        with_type(dtype, [&](auto o) {
            using OT = decltype(o);
            if (h->cfg.state_bits == 8)
                adamw_moments_kernel<OT, true><<<grid, 256, 0, stream()>>>(h->args(), h->total, (OT *)m_dev, (OT *)v_dev);
            else
                adamw_moments_kernel<OT, false><<<grid, 256, 0, stream()>>>(h->args(), h->total, (OT *)m_dev, (OT *)v_dev);
        });
        launch_check("adamw_moments_kernel");
    });
}

extern "C" int snk_adamw_get_steps(snk_adamw h, int64_t *steps) {
    return guard([&] {
        SNK_CHECK(h && steps, SNK_ERR_INVALID, "NULL argument");
        check_device(h);
        adamw_not_captured(stream(), "the step count is read");
        AdamCtl ctl{};
        SNK_HIP(hipMemcpyAsync(&ctl, h->ctl.p, sizeof ctl, hipMemcpyDeviceToHost, stream()));
        SNK_HIP(hipStreamSynchronize(stream()));
        *steps = ctl.t - (ctl.skip ? 1 : 0);
    });
}

extern "C" int snk_adamw_set_steps(snk_adamw h, int64_t steps) {
    return guard([&] {
        SNK_CHECK(h && steps >= 0, SNK_ERR_INVALID, "bad adamw_set_steps arguments");
        check_device(h);
        adamw_not_captured(stream(), "the step count is set");
        AdamCtl ctl{};
        ctl.t = steps;
        ctl.c1 = 1.0 - std::pow(h->cfg.beta1, (double)steps);
        ctl.c2 = 1.0 - std::pow(h->cfg.beta2, (double)steps);
        h->now = AdamStep{steps, ctl.c1, ctl.c2, 0.0f, 0.0f};
        static_assert(offsetof(AdamCtl, norm) == 28, "t, c1, c2 and skip lead the struct");
        SNK_HIP(hipMemcpyAsync(h->ctl.p, &ctl, offsetof(AdamCtl, norm), hipMemcpyHostToDevice, stream()));
        SNK_HIP(hipStreamSynchronize(stream()));
    });
}
