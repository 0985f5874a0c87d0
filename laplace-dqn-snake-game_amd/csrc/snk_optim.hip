// snk_optim.hip — AdamW over a list of tensors (include/snakehip.h), moments in 32 bits or in
// 8-bit codes with block scales.
//
// The step moves 28 B per fp32 element (p, m, v read and written, g read; 8-bit moments: 16 B) for
// ~20 operations, so HBM bounds it: every tensor is cut into chunks of CH elements, a table names
// each chunk's tensor, and one launch covers all tensors, whatever their number and sizes. A wave
// owns 256 consecutive elements (the 8-bit block), a lane four of them: 16-byte accesses, and the
// block's two scales are one wave reduction each.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <vector>

#include "snk_optim.hpp"

namespace snk {

constexpr int BLK = 256;        // elements of a wave's block = the 8-bit states' block
constexpr int CH = 4096;        // elements of a workgroup's chunk (a multiple of 4 BLK)
constexpr int NORM_WG = 1024;   // most workgroups (= partial sums) of the norm pass

struct AdamTensor {
    void *p, *c;          // parameters, their rounded copy (or nullptr)
    const void *g;
    int64_t size, start;  // elements, first place in the state layout
    float wd;
    int32_t pad;
};
struct AdamChunk {
    int32_t tensor, index;   // elements [index * CH, ...) of the tensor
};
struct alignas(16) AdamCtl {
    int64_t t;            // steps taken
    float norm;           // N of the last step
    float gmul;           // s c of the step under way
    float ibc1, ibc2;     // 1 / (1 - b^t)
    int32_t skip;         // N was not finite
    int32_t pad;
};
struct AdamHyper {
    double b1d, b2d;
    float b1, omb1, b2, omb2, eps, lr, gscale, max_norm;
    int32_t copy_dtype;
    uint64_t seed;
};

// four consecutive elements at an element-aligned address: one 16- or 8-byte access (unaligned
// global accesses are legal on gfx950), so views that start anywhere take the same path
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) pack4 {
    T v[4];
};
template <class T>
__device__ __forceinline__ void load4(const T *p, int64_t i, int64_t n, float *x) {
    if (i + 4 <= n) {
        const pack4<T> q = *reinterpret_cast<const pack4<T> *>(p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (float)q.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = i + k < n ? (float)p[i + k] : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store4(T *p, int64_t i, int64_t n, const float *x) {
    if (i + 4 <= n) {
        pack4<T> q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q.v[k] = (T)x[k];   // round to nearest even
        *reinterpret_cast<pack4<T> *>(p + i) = q;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) p[i + k] = (T)x[k];
    }
}

// largest of 64 non-negative floats (0 where a lane has no partner)
__device__ __forceinline__ float wave_max_nonneg(float x) {
    auto step = [&](auto ctrl, auto mask) {
        const float y = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value,
                                                                   decltype(mask)::value, 0xf, false));
        x = fmaxf(x, y);
    };
    step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});   // row_shr 1, 2, 4, 8
    step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});   // row_bcast 15, 31
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// the values the 8-bit codes stand for
__device__ __forceinline__ float m_value(int a, float scale) {
    return (float)(a * abs(a)) * (1.0f / 16129.0f) * scale;
}
__device__ __forceinline__ float v_level(float b) {   // (b / 255)^4, b^2 exact
    const float b2 = b * b;
    return (b2 * b2) * (1.0f / 4228250625.0f);
}

// partial sums of (s g)^2 in fp64: fp32 squares overflow above 1.8e19 and lose the small ones
template <class GT>
__global__ __launch_bounds__(256) void adamw_norm_kernel(const AdamTensor *__restrict__ tab,
                                                         const AdamChunk *__restrict__ chunks, int64_t n_chunks,
                                                         float gscale, double *__restrict__ part) {
    __shared__ double sh[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double sum = 0.0;
    for (int64_t c = blockIdx.x; c < n_chunks; c += gridDim.x) {
        const AdamChunk k = chunks[c];
        const AdamTensor T = tab[k.tensor];
        const int64_t base = (int64_t)k.index * CH + wave * BLK + lane * 4;
#pragma unroll
        for (int j = 0; j < CH / (4 * BLK); ++j) {
            const int64_t i = base + j * 4 * BLK;
            if (i >= T.size) break;
            float g[4];
            load4((const GT *)T.g, i, T.size, g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double d = (double)(g[e] * gscale);
                sum = fma(d, d, sum);
            }
        }
    }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) sh[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// the step's scalars, once: N and the clip factor from the partial sums, the bias corrections in
// fp64 (1 - b^t loses digits in fp32 while t is small), the step count
__global__ __launch_bounds__(256) void adamw_begin_kernel(AdamCtl *__restrict__ ctl, const double *__restrict__ part,
                                                          int n_part, AdamHyper H) {
    __shared__ double sh[256];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n_part; i += 256) sum += part[i];
    sh[threadIdx.x] = sum;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    float gmul = H.gscale;
    if (n_part > 0) {
        const double N = sqrt(sh[0]);
        ctl->norm = (float)N;
        const bool fine = N < INFINITY;   // false for NaN too
        ctl->skip = fine ? 0 : 1;
        if (!fine) return;
        if (N > (double)H.max_norm) gmul = (float)((double)H.gscale * ((double)H.max_norm / N));
    }
    const int64_t t = ctl->t + 1;
    ctl->t = t;
    ctl->gmul = gmul;
    ctl->ibc1 = (float)(1.0 / (1.0 - pow(H.b1d, (double)t)));
    ctl->ibc2 = (float)(1.0 / (1.0 - pow(H.b2d, (double)t)));
}

struct AdamArgs {
    const AdamTensor *tab;
    const AdamChunk *chunks;
    void *m, *v;
    float *ms, *vs;
    const AdamCtl *ctl;
    AdamHyper H;
};

// one element: new moments in m, v; the new parameter is returned
__device__ __forceinline__ float adamw_one(const AdamHyper &H, float gmul, float ibc1, float ibc2, float wd, float p,
                                           float g, float &m, float &v) {
    g *= gmul;
    m = H.b1 * m + H.omb1 * g;
    v = H.b2 * v + H.omb2 * (g * g);
    const float step = (m * ibc1) / (__builtin_sqrtf(v * ibc2) + H.eps);
    return p - H.lr * (step + wd * p);
}

template <class PT>
__device__ __forceinline__ void store_params(const AdamTensor &T, int copy_dtype, int64_t i, const float *p) {
    store4((PT *)T.p, i, T.size, p);
    if (T.c) {
        if (copy_dtype == SNK_BF16)
            store4((__bf16 *)T.c, i, T.size, p);
        else
            store4((_Float16 *)T.c, i, T.size, p);
    }
}

template <class PT, class GT>
__global__ __launch_bounds__(256) void adamw32_kernel(AdamArgs A) {
    if (A.ctl->skip) return;
    const float gmul = A.ctl->gmul, ibc1 = A.ctl->ibc1, ibc2 = A.ctl->ibc2;
    const AdamChunk k = A.chunks[blockIdx.x];
    const AdamTensor T = A.tab[k.tensor];
    const int64_t base = (int64_t)k.index * CH + threadIdx.x * 4;
    float *ms = (float *)A.m + T.start, *vs = (float *)A.v + T.start;
#pragma unroll
    for (int j = 0; j < CH / (4 * BLK); ++j) {
        const int64_t i = base + j * 4 * BLK;
        if (i >= T.size) break;
        float p[4], g[4];
        load4((const PT *)T.p, i, T.size, p);
        load4((const GT *)T.g, i, T.size, g);
        float4 m = *(float4 *)(ms + i), v = *(float4 *)(vs + i);   // padded: always whole
        p[0] = adamw_one(A.H, gmul, ibc1, ibc2, T.wd, p[0], g[0], m.x, v.x);
        p[1] = adamw_one(A.H, gmul, ibc1, ibc2, T.wd, p[1], g[1], m.y, v.y);
        p[2] = adamw_one(A.H, gmul, ibc1, ibc2, T.wd, p[2], g[2], m.z, v.z);
        p[3] = adamw_one(A.H, gmul, ibc1, ibc2, T.wd, p[3], g[3], m.w, v.w);
        *(float4 *)(ms + i) = m;
        *(float4 *)(vs + i) = v;
        store_params<PT>(T, A.H.copy_dtype, i, p);
    }
}

template <class PT, class GT>
__global__ __launch_bounds__(256) void adamw8_kernel(AdamArgs A) {
    if (A.ctl->skip) return;
    const float gmul = A.ctl->gmul, ibc1 = A.ctl->ibc1, ibc2 = A.ctl->ibc2;
    const AdamChunk k = A.chunks[blockIdx.x];
    const AdamTensor T = A.tab[k.tensor];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t key = splitmix64(A.H.seed ^ ((uint64_t)A.ctl->t * 0xD1B54A32D192ED03ULL));   // rng_hash's first half
#pragma unroll
    for (int j = 0; j < CH / (4 * BLK); ++j) {
        const int64_t first = (int64_t)k.index * CH + (j * 4 + wave) * BLK;   // the wave's block
        if (first >= T.size) break;
        const int64_t i = first + lane * 4, place = T.start + i, block = (T.start + first) / BLK;
        float p[4], g[4], m[4], v[4];
        load4((const PT *)T.p, i, T.size, p);
        load4((const GT *)T.g, i, T.size, g);
        const uint32_t mc = *(const uint32_t *)((const uint8_t *)A.m + place);
        const uint32_t vc = *(const uint32_t *)((const uint8_t *)A.v + place);
        const float ms0 = A.ms[block], vs0 = A.vs[block];
        float mmax = 0.0f, vmax = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {   // places behind the tensor's end hold zeros and read g = 0
            m[e] = m_value((int)(int8_t)(mc >> (8 * e)), ms0);
            v[e] = v_level((float)((vc >> (8 * e)) & 255u)) * vs0;
            p[e] = adamw_one(A.H, gmul, ibc1, ibc2, T.wd, p[e], g[e], m[e], v[e]);
            mmax = fmaxf(mmax, fabsf(m[e]));
            vmax = fmaxf(vmax, v[e]);
        }
        store_params<PT>(T, A.H.copy_dtype, i, p);
        mmax = wave_max_nonneg(mmax);
        vmax = wave_max_nonneg(vmax);
        const uint64_t h = splitmix64(key ^ (uint64_t)(place >> 2));
        uint32_t mo = 0, vo = 0;
        const float im = mmax > 0.0f ? mmax : 1.0f, iv = vmax > 0.0f ? vmax : 1.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int a = (int)rintf(127.0f * __builtin_sqrtf(fabsf(m[e]) / im));
            mo |= (uint32_t)((m[e] < 0.0f ? -a : a) & 255) << (8 * e);
            const float part = v[e] / iv;
            const float low = fminf(floorf(255.0f * __builtin_sqrtf(__builtin_sqrtf(part))), 254.0f);
            const float lo = v_level(low), hi = v_level(low + 1.0f);
            const float r = (float)((uint32_t)(h >> (16 * e)) & 0xFFFFu);
            uint32_t b = (uint32_t)low + (r < (part - lo) / (hi - lo) * 65536.0f ? 1u : 0u);
            if (v[e] > 0.0f && b == 0) b = 1;   // never back as 0: m / eps would follow
            vo |= (b & 255u) << (8 * e);
        }
        *(uint32_t *)((uint8_t *)A.m + place) = mo;
        *(uint32_t *)((uint8_t *)A.v + place) = vo;
        if (lane == 0) {
            A.ms[block] = mmax;
            A.vs[block] = vmax;
        }
    }
}

// the moments' values, a lane four places
template <class OT, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_moments_kernel(AdamArgs A, int64_t total, OT *__restrict__ mo,
                                                            OT *__restrict__ vo) {
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < total; i += (int64_t)gridDim.x * 1024) {
        float m[4], v[4];
        if (EIGHT) {
            const uint32_t mc = *(const uint32_t *)((const uint8_t *)A.m + i);
            const uint32_t vc = *(const uint32_t *)((const uint8_t *)A.v + i);
            const float ms = A.ms[i / BLK], vs = A.vs[i / BLK];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = m_value((int)(int8_t)(mc >> (8 * e)), ms);
                v[e] = v_level((float)((vc >> (8 * e)) & 255u)) * vs;
            }
        } else {
            load4((const float *)A.m, i, total, m);
            load4((const float *)A.v, i, total, v);
        }
        if (mo) store4(mo, i, total, m);
        if (vo) store4(vo, i, total, v);
    }
}

// tensor addresses into the device table, by value: safe inside a capture, where a host array
// would be read again at every replay
constexpr int BIND_N = 128;
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
__global__ void adamw_fill_kernel(uint32_t *__restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = 0;
}

}  // namespace snk

using namespace snk;

struct snk_adamw_s {
    snk_adamw_cfg_t cfg{};
    int device = 0;
    bool owned = false, bound = false;
    std::vector<int64_t> size, start;
    int64_t total = 0, n_chunks = 0;
    DevBuf<AdamTensor> tab;
    DevBuf<AdamChunk> chunks;
    DevBuf<uint8_t> m, v;
    DevBuf<float> ms, vs;
    DevBuf<double> part;
    DevBuf<AdamCtl> ctl;
    int64_t state_bytes() const { return total * (cfg.state_bits / 8); }
    AdamArgs args() const {
        AdamArgs a{};
        a.tab = tab.p;
        a.chunks = chunks.p;
        a.m = m.p;
        a.v = v.p;
        a.ms = ms.p;
        a.vs = vs.p;
        a.ctl = ctl.p;
        return a;
    }
};

static int dtype_size(int32_t d) { return d == SNK_F32 ? 4 : 2; }
static bool dtype_ok(int32_t d) { return d == SNK_F32 || d == SNK_BF16 || d == SNK_F16; }

static void check_device(snk_adamw h) {
    int dev = 0;
    SNK_HIP(hipGetDevice(&dev));
    SNK_CHECK(dev == h->device, SNK_ERR_STATE, "the AdamW handle lives on device %d, the current device is %d", h->device,
              dev);
}

namespace snk {

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
    SNK_CHECK(cfg->eps > 0 && (float)cfg->eps > 0 && cfg->eps < INFINITY, SNK_ERR_INVALID,
              "AdamW: eps %g is not a positive fp32 number", cfg->eps);
    SNK_CHECK(cfg->max_grad_norm >= 0, SNK_ERR_INVALID, "AdamW: max_grad_norm %g is negative", cfg->max_grad_norm);
    SNK_CHECK(cfg->reserved == 0, SNK_ERR_INVALID, "AdamW: reserved must be 0");
    auto h = std::make_unique<snk_adamw_s>();
    h->cfg = *cfg;
    SNK_HIP(hipGetDevice(&h->device));
    std::vector<AdamTensor> tab(n);
    std::vector<AdamChunk> chunks;
    for (int i = 0; i < n; ++i) {
        SNK_CHECK(sizes[i] >= 0 && sizes[i] < (int64_t)1 << 40 && h->total < (int64_t)1 << 40, SNK_ERR_INVALID,
                  "AdamW: tensor %d has %lld elements", i, (long long)sizes[i]);
        SNK_CHECK(wd[i] >= 0 && wd[i] < INFINITY, SNK_ERR_INVALID, "AdamW: weight decay %g of tensor %d", wd[i], i);
        h->size.push_back(sizes[i]);
        h->start.push_back(h->total);
        tab[i] = AdamTensor{nullptr, nullptr, nullptr, sizes[i], h->total, wd[i], 0};
        for (int64_t c = 0; c * CH < sizes[i]; ++c) chunks.push_back(AdamChunk{i, (int32_t)c});
        h->total += (sizes[i] + BLK - 1) / BLK * BLK;
    }
    h->n_chunks = (int64_t)chunks.size();
    SNK_CHECK(h->n_chunks < (int64_t)1 << 31, SNK_ERR_INVALID, "AdamW: too many elements for one handle");
    h->tab = DevBuf<AdamTensor>(n);
    h->chunks = DevBuf<AdamChunk>(chunks.size());
    h->m = DevBuf<uint8_t>(h->state_bytes());
    h->v = DevBuf<uint8_t>(h->state_bytes());
    if (cfg->state_bits == 8) {
        h->ms = DevBuf<float>(h->total / BLK);
        h->vs = DevBuf<float>(h->total / BLK);
    }
    h->part = DevBuf<double>(NORM_WG);
    h->ctl = DevBuf<AdamCtl>(1);
    hipStream_t s = stream();
    SNK_HIP(hipMemcpyAsync(h->tab, tab.data(), n * sizeof(AdamTensor), hipMemcpyHostToDevice, s));
    if (!chunks.empty())
        SNK_HIP(hipMemcpyAsync(h->chunks, chunks.data(), chunks.size() * sizeof(AdamChunk), hipMemcpyHostToDevice, s));
    adamw_reset(h.get(), s);
    SNK_HIP(hipStreamSynchronize(s));
    return h.release();
}

void adamw_free(snk_adamw h) { delete h; }
void adamw_set_owned(snk_adamw h) { h->owned = true; }

void adamw_bind(snk_adamw h, void *const *params, const void *const *grads, void *const *copies, hipStream_t s) {
    const int n = (int)h->size.size();
    SNK_CHECK(params && grads, SNK_ERR_INVALID, "adamw_bind: NULL argument");
    SNK_CHECK((copies != nullptr) == (h->cfg.copy_dtype >= 0), SNK_ERR_INVALID,
              "adamw_bind: copies go with a copy_dtype, and only with one");
    struct Span {
        uintptr_t lo, hi;
        bool written;
    };
    std::vector<Span> spans;
    auto add = [&](const void *p, int i, int32_t dtype, bool written, const char *what) {
        if (h->size[i] == 0) return;
        const uintptr_t a = reinterpret_cast<uintptr_t>(p);
        SNK_CHECK(a && a % dtype_size(dtype) == 0, SNK_ERR_INVALID, "adamw_bind: %s %d is NULL or not element-aligned",
                  what, i);
        spans.push_back(Span{a, a + (uintptr_t)h->size[i] * dtype_size(dtype), written});
    };
    for (int i = 0; i < n; ++i) {
        add(params[i], i, h->cfg.param_dtype, true, "parameter");
        add(grads[i], i, h->cfg.grad_dtype, false, "gradient");
        if (copies) add(copies[i], i, h->cfg.copy_dtype, true, "copy");
    }
    // a tensor that is written must not overlap any other: the chunks run in no order. Swept by
    // address with the furthest end seen of all spans and of the written ones
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
    uintptr_t end = 0, end_written = 0;
    for (const Span &x : spans) {
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
            b.g[i] = grads[at + i];
            b.c[i] = copies ? copies[at + i] : nullptr;
        }
        adamw_bind_kernel<<<1, BIND_N, 0, s>>>(h->tab + at, b, k);
        launch_check("adamw_bind_kernel");
    }
    h->bound = true;
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

void adamw_step(snk_adamw h, float lr, float grad_scale, hipStream_t s) {
    SNK_CHECK(h->bound, SNK_ERR_STATE, "AdamW: no tensors are bound");
    SNK_CHECK(lr >= 0 && lr < INFINITY && std::isfinite(grad_scale), SNK_ERR_INVALID, "AdamW: lr %g, grad_scale %g", lr,
              grad_scale);
    const snk_adamw_cfg_t &c = h->cfg;
    AdamArgs A = h->args();
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
    int n_part = 0;
    if (c.max_grad_norm > 0) {
        n_part = (int)std::max<int64_t>(1, std::min<int64_t>(h->n_chunks, NORM_WG));
        with_type(c.grad_dtype, [&](auto g) {
            adamw_norm_kernel<decltype(g)><<<n_part, 256, 0, s>>>(h->tab, h->chunks, h->n_chunks, grad_scale, h->part);
        });
        launch_check("adamw_norm_kernel");
    }
    adamw_begin_kernel<<<1, 256, 0, s>>>(h->ctl, h->part, n_part, H);
    launch_check("adamw_begin_kernel");
    if (h->n_chunks == 0) return;
    with_type(c.param_dtype, [&](auto p) {
        with_type(c.grad_dtype, [&](auto g) {
            using PT = decltype(p);
            using GT = decltype(g);
            if (c.state_bits == 8)
                adamw8_kernel<PT, GT><<<(unsigned)h->n_chunks, 256, 0, s>>>(A);
            else
                adamw32_kernel<PT, GT><<<(unsigned)h->n_chunks, 256, 0, s>>>(A);
        });
    });
    launch_check("adamw_kernel");
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
        (void)hipStreamSynchronize(stream());
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
        SNK_HIP(hipMemcpyAsync(steps, &h->ctl.p->t, sizeof *steps, hipMemcpyDeviceToHost, stream()));
        SNK_HIP(hipStreamSynchronize(stream()));
    });
}

extern "C" int snk_adamw_set_steps(snk_adamw h, int64_t steps) {
    return guard([&] {
        SNK_CHECK(h && steps >= 0, SNK_ERR_INVALID, "bad adamw_set_steps arguments");
        check_device(h);
        SNK_HIP(hipMemcpyAsync(&h->ctl.p->t, &steps, sizeof steps, hipMemcpyHostToDevice, stream()));
        SNK_HIP(hipStreamSynchronize(stream()));
    });
}
