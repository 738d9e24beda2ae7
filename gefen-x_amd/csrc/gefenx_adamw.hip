// gefenx_adamw.hip -- AdamW over many tensors, its moments in fp32 or in 8 bits.
//
//   m <- b1 m + (1-b1) g,  v <- b2 v + (1-b2) g^2        (g scaled by the clip coefficient)
//   p <- p (1 - lr wd) - lr/bc1 * m / (sqrt(v) / sqrt(bc2) + eps)
//
// All of it is one pass over memory: a few operations an element against 22 bytes (bf16, fp32 moments)
// or 10 (8-bit moments).  Descriptors of up to kItems tensors travel in the kernel's arguments, so a step
// uploads nothing and a launch covers many tensors; workgroups find theirs by the running workgroup count.
#include <hip/hip_runtime.h>

#include "gefenx.h"
#include "gefenx_device.h"
#include "gefenx_internal.h"
#include "gefenx_run.h"

namespace gx {
namespace {

constexpr int kT = 256;                  // threads of a workgroup
constexpr int kItems = 36;               // tensors of a launch: 36 * 108 bytes of kernel arguments
constexpr int kBlock8 = 256;             // elements per scale of the 8-bit moments
constexpr int kGroup = 16;               // lanes that share such a block, 16 elements each
constexpr float kTiny = 0x1p-126f;       // smallest scale: its reciprocal, and 448 of them, are finite
constexpr int kCode0 = 761;              // bits(x) >> 20 of v's code c is c + 761: code 255 is x = 1
constexpr int64_t kNormPartials = 4096;  // about so many partial sums of the gradient norm
// A launch has fewer than 2^32 threads; a tensor has its workgroups in one.
constexpr int64_t kMaxWgs = ((int64_t)1 << 32) / kT - 1, kMaxNumel = (int64_t)1 << 33;

struct Item {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* vs;
    int64_t n;
    uint64_t key;
    float step, wdf, b1, a1, b2, a2, rbc2, eps;
    const gefenx_adamw_row* row;  // captured steps: where step, wdf, rbc2 and key are
};

// What of an Item changes from step to step.
struct Scalars {
    float step, wdf, rbc2;
    uint64_t key;
};
__device__ __forceinline__ Scalars scalars_of(const Item& t) {
    if (!t.row) return Scalars{t.step, t.wdf, t.rbc2, t.key};
    return Scalars{sload(&t.row->step_size), sload(&t.row->wd_factor), sload(&t.row->inv_sqrt_bc2), sload(&t.row->key)};
}

struct Batch {
    Item it[kItems];
    int32_t end[kItems];  // workgroups up to and including tensor i
    int32_t n;
    int32_t iters;        // gradient norm: passes of a workgroup
};
static_assert(sizeof(Batch) <= 4080, "kernel arguments");

// The tensor of workgroup w, and w's place within it.
__device__ __forceinline__ int find_item(const Batch& b, int w, int& local) {
    int lo = 0, hi = b.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (w < b.end[mid]) hi = mid; else lo = mid + 1;
    }
    local = lo ? w - b.end[lo - 1] : w;
    return lo;
}

// ------------------------------------------------------------ runs of elements
// A lane moves W consecutive elements at a time: 16 bytes of the widest stream beside it, so that a
// wave's accesses to that stream leave no gaps (two 16-byte pieces of 8 fp32 elements a lane took the
// fp32 step of 218M bf16 elements from 793 to 883 us).  Whole runs by vector accesses of any
// alignment, a tensor's last one by elements.

// Four codes to a word.
__device__ __forceinline__ uint32_t load_codes4(const uint8_t* base, int64_t left) {
    typedef uint32_t V __attribute__((aligned(1)));
    if (left >= 4) return __builtin_nontemporal_load(GX_GLOBAL_AS(const V, base));
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 3; ++k)
        if (k < left) w |= (uint32_t)*gbl(base + k) << (8 * k);
    return w;
}

template <int W>
__device__ __forceinline__ void load_codes(const uint8_t* base, int64_t left, uint32_t (&c)[W / 4]) {
    if (W == 8 && left >= 8) {
        const RawIdx8 v = load_raw_idx8_any(base);
        c[0] = v.lo;
        c[W / 4 - 1] = v.hi;
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) c[i] = load_codes4(base + 4 * i, left - 4 * i);
    }
}

template <int W>
__device__ __forceinline__ void store_codes(uint8_t* base, int64_t left, const uint32_t (&c)[W / 4]) {
    if (left >= W) {
        if constexpr (W == 8) {
            const u32x2 a = {c[0], c[1]};
            __builtin_nontemporal_store(a, GX_GLOBAL_AS(u32x2_a1, base));
        } else {
            typedef uint32_t V __attribute__((aligned(1)));
            __builtin_nontemporal_store(c[0], GX_GLOBAL_AS(V, base));
        }
    } else {
#pragma unroll
        for (int k = 0; k < W; ++k)
            if (k < left) *gbl(base + k) = (uint8_t)(c[k >> 2] >> (8 * (k & 3)));
    }
}

// The moments round after each operation, as the formula written in torch does, so 8-bit codes follow
// from the inputs alone.
__device__ __forceinline__ void advance(const Item& t, float g, float& m, float& v) {
    m = m * t.b1 + g * t.a1;
    v = v * t.b2 + g * g * t.a2;
}
// FAST: the hardware's square root and reciprocal, 1 unit each, as good as the exact ones before p
// rounds.  That square root takes v below 2^-126 for 0, which eps has to drown: drowns().
template <bool FAST>
__device__ __forceinline__ float stepped(const Scalars& s, float eps, float p, float m, float v) {
    if constexpr (FAST) {
        const float d = __builtin_fmaf(__builtin_amdgcn_sqrtf(v), s.rbc2, eps);
        return __builtin_fmaf(-s.step, m * __builtin_amdgcn_rcpf(d), p * s.wdf);
    } else {
        const float d = __builtin_fmaf(__builtin_sqrtf(v), s.rbc2, eps);
        return __builtin_fmaf(-s.step, m / d, p * s.wdf);
    }
}

// ------------------------------------------------------------ fp32 moments
// 22 bytes an element (bf16): 218M elements 785-817 us, 5.9-6.1 TB/s, where a copy of 2 GiB reaches 5.8.
constexpr int kW32 = 4;  // elements of a lane
template <int DT>
__global__ __launch_bounds__(kT) void k_adamw(const Batch b, const float* __restrict__ coef) {
    using T = typename Elem<DT>::T;
    int local;
    const Item& t = b.it[find_item(b, (int)blockIdx.x, local)];
    const Scalars sc = scalars_of(t);
    const float c = coef ? sload(coef) : 1.0f;
    const int64_t at = ((int64_t)local * kT + threadIdx.x) * kW32;
    const int64_t left = t.n - at;
    if (left <= 0) return;
    const auto g = load_run<T, kW32>((const T*)t.g + at, left);
    auto m = load_run<float, kW32>((const float*)t.m + at, left), v = load_run<float, kW32>((const float*)t.v + at, left);
    auto p = load_run<T, kW32>((const T*)t.p + at, left);
#pragma unroll
    for (int k = 0; k < kW32; ++k) {
        advance(t, to_f32<DT>(g.e[k]) * c, m.e[k], v.e[k]);
        p.e[k] = from_f32<DT>(stepped<false>(sc, t.eps, to_f32<DT>(p.e[k]), m.e[k], v.e[k]));
    }
    store_run<float, kW32>((float*)t.m + at, left, m);
    store_run<float, kW32>((float*)t.v + at, left, v);
    store_run<T, kW32>((T*)t.p + at, left, p);
}

// ------------------------------------------------------------ 8-bit moments
// m: E4M3 (the hardware's conversions, nearest even), scale = largest |m| / 448.
// v: 5 exponent and 3 mantissa bits of v / (largest v), code 0 for zero alone, so that an element
// whose v is far below its block's is held too large, never at zero (its step is m / sqrt(v)).  A
// step moves v by a share of about 1 - b2, far less than half a code, so nearest rounding would
// hold it where it is: the cut bits are rounded up with their own probability instead, by 16 bits
// of a counter generator.

__device__ __forceinline__ uint64_t mix64(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ULL;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBULL;
    return z ^ (z >> 31);
}

__device__ __forceinline__ void decode_m(uint32_t c, float scale, float* m) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    m[0] = a[0] * scale; m[1] = a[1] * scale; m[2] = b[0] * scale; m[3] = b[1] * scale;
}

__device__ __forceinline__ void decode_v(uint32_t c, float scale, float* v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t x = (c >> (8 * k)) & 0xffu;
        v[k] = (x ? __uint_as_float((x + kCode0) << 20) : 0.0f) * scale;
    }
}

__device__ __forceinline__ uint32_t encode_m(const float* m, float inv) {
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __builtin_amdgcn_fmed3f(m[k] * inv, -448.0f, 448.0f);
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
}

// at: the first element of the four, a multiple of 4: one draw
__device__ __forceinline__ uint32_t encode_v(const float* v, float inv, uint64_t key, int64_t at) {
    const uint64_t z = mix64(key + 0x9E3779B97F4A7C15ULL * ((uint64_t)(at >> 2) + 1));
    const uint32_t r[2] = {(uint32_t)z, (uint32_t)(z >> 32)};
    uint32_t packed = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t dither = (k & 1 ? r[k >> 1] >> 12 : r[k >> 1] << 4) & 0xffff0u;
        int c = (int)((__float_as_uint(v[k] * inv) + dither) >> 20) - kCode0;
        c = c < 1 ? 1 : (c > 255 ? 255 : c);
        packed |= (uint32_t)(v[k] == 0.0f ? 0 : c) << (8 * k);
    }
    return packed;
}

// Largest value of a block's 16 lanes, in each of them (bits of non-negative floats, NaN above inf).
__device__ __forceinline__ uint32_t group16_max(uint32_t v) {
    uint32_t o;
    o = dpp32<0xB1, 0xf>(v); v = o > v ? o : v;
    o = dpp32<0x4E, 0xf>(v); v = o > v ? o : v;
    o = dpp32<0x141, 0xf>(v); v = o > v ? o : v;
    o = dpp32<0x140, 0xf>(v); return o > v ? o : v;
}

// A block that holds an inf or NaN gets the scale NaN: all of it reads as NaN from then on.
__device__ __forceinline__ float block_scale(float amax) {
    return amax <= 3.402823466e38f ? (amax > kTiny ? amax : kTiny) : __uint_as_float(0x7fc00000u);
}

// A block of 256 elements by 16 lanes, each with N runs of W of them: the moments stay in registers
// between the block's maxima and its codes, and the maxima cross lanes within a DPP row.  10.06 bytes an
// element (bf16): 1.05e9 elements 1.80 ms, 5.9 TB/s; with the exact square root and division the
// arithmetic takes longer than the memory (218M elements 368 -> 523 us).
template <int DT, bool FAST>
__global__ __launch_bounds__(kT) void k_adamw8(const Batch b, const float* __restrict__ coef) {
    using T = typename Elem<DT>::T;
    constexpr int W = 16 / sizeof(T), N = kBlock8 / (kGroup * W);
    int local;
    const Item& t = b.it[find_item(b, (int)blockIdx.x, local)];
    const Scalars sc = scalars_of(t);
    const float c = coef ? sload(coef) : 1.0f;
    const int lane = threadIdx.x & (kGroup - 1);
    const int64_t blk = (int64_t)local * (kT / kGroup) + threadIdx.x / kGroup;
    // the 16 lanes of a block leave together or stay together: what they exchange is among themselves
    if (blk * kBlock8 >= t.n) return;
    const int64_t at0 = blk * kBlock8 + lane * W;
    Run<T, W> g[N], p[N];
    uint32_t mc[N][W / 4], vc[N][W / 4];
    const float ms = *gbl(t.ms + blk), vs = *gbl(t.vs + blk);
#pragma unroll
    for (int h = 0; h < N; ++h) {
        const int64_t at = at0 + h * kGroup * W, left = t.n - at;
        g[h] = load_run<T, W>((const T*)t.g + at, left);
        load_codes<W>((const uint8_t*)t.m + at, left, mc[h]);
        load_codes<W>((const uint8_t*)t.v + at, left, vc[h]);
        p[h] = load_run<T, W>((const T*)t.p + at, left);
    }
    float m[N][W], v[N][W];
    uint32_t mx = 0, vx = 0;
#pragma unroll
    for (int h = 0; h < N; ++h) {
        const int64_t at = at0 + h * kGroup * W, left = t.n - at;
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            decode_m(mc[h][i], ms, m[h] + 4 * i);
            decode_v(vc[h][i], vs, v[h] + 4 * i);
        }
#pragma unroll
        for (int k = 0; k < W; ++k) {
            advance(t, to_f32<DT>(g[h].e[k]) * c, m[h][k], v[h][k]);
            p[h].e[k] = from_f32<DT>(stepped<FAST>(sc, t.eps, to_f32<DT>(p[h].e[k]), m[h][k], v[h][k]));
            const uint32_t mb = __float_as_uint(m[h][k]) & 0x7fffffffu, vb = __float_as_uint(v[h][k]) & 0x7fffffffu;
            mx = mb > mx ? mb : mx;
            vx = vb > vx ? vb : vx;
        }
        store_run<T, W>((T*)t.p + at, left, p[h]);
    }
    const float mscale = block_scale(__uint_as_float(group16_max(mx)) * (1.0f / 448.0f));
    const float vscale = block_scale(__uint_as_float(group16_max(vx)));
    const float minv = 1.0f / mscale, vinv = 1.0f / vscale;
#pragma unroll
    for (int h = 0; h < N; ++h) {
        const int64_t at = at0 + h * kGroup * W, left = t.n - at;
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            mc[h][i] = encode_m(m[h] + 4 * i, minv);
            vc[h][i] = encode_v(v[h] + 4 * i, vinv, sc.key, at + 4 * i);
        }
        store_codes<W>((uint8_t*)t.m + at, left, mc[h]);
        store_codes<W>((uint8_t*)t.v + at, left, vc[h]);
    }
    if (lane == 0) {
        *gbl(t.ms + blk) = mscale;
        *gbl(t.vs + blk) = vscale;
    }
}

// The values that 8-bit moments stand for: Item::p and Item::g are where m's and v's go.  Mostly writes:
// 1.05e9 elements 1.68 ms, 6.3 TB/s.
__global__ __launch_bounds__(kT) void k_adamw8_values(const Batch b) {
    int local;
    const Item& t = b.it[find_item(b, (int)blockIdx.x, local)];
    const int64_t at = ((int64_t)local * kT + threadIdx.x) * 4;
    const int64_t left = t.n - at;
    if (left <= 0) return;
    const uint32_t mc = load_codes4((const uint8_t*)t.m + at, left), vc = load_codes4((const uint8_t*)t.v + at, left);
    const int64_t blk = at / kBlock8;
    Run<float, 4> x;
    decode_m(mc, *gbl(t.ms + blk), x.e);
    store_run<float, 4>((float*)t.p + at, left, x);
    decode_v(vc, *gbl(t.vs + blk), x.e);
    store_run<float, 4>((float*)const_cast<void*>(t.g) + at, left, x);
}

// ------------------------------------------------------------ gradient norm
// Sums of squares in float64, one partial per workgroup, added up by one workgroup in a fixed order.  One
// read of the gradients: 436 MB 67-77 us, 5.7-6.5 TB/s (a read alone reaches 7.1).  Ordinary loads, not streamed
// ones: the step that follows finds part of them in the 256 MB cache (both 884 -> 851 us, with 8-bit
// moments 448 -> 421; 92M elements 355 -> 335).
template <int DT>
__global__ __launch_bounds__(kT) void k_grad_sumsq(const Batch b, double* __restrict__ partials) {
    using T = typename Elem<DT>::T;
    __shared__ double waves[kT / 64];
    int local;
    const Item& t = b.it[find_item(b, (int)blockIdx.x, local)];
    double s = 0.0;
    for (int it = 0; it < b.iters; ++it) {
        const int64_t at = (((int64_t)local * b.iters + it) * kT + threadIdx.x) * 8;
        const int64_t left = t.n - at;
        if (left <= 0) break;
        const auto g = load_run<T, 8, false>((const T*)t.g + at, left);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const double x = (double)to_f32<DT>(g.e[k]);
            s = __builtin_fma(x, x, s);
        }
    }
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = waves[0];
        for (int w = 1; w < kT / 64; ++w) total += waves[w];
        *gbl(partials + blockIdx.x) = total;
    }
}

__global__ __launch_bounds__(1024) void k_grad_norm(const double* __restrict__ partials, int64_t n, double max_norm,
                                                    float* __restrict__ out) {
    __shared__ double waves[16];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += *gbl(partials + i);
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = waves[0];
        for (int w = 1; w < 16; ++w) total += waves[w];
        const float norm = (float)sqrt(total);
        const float c = (float)max_norm / (norm + 1e-6f);
        out[0] = norm;
        out[1] = c >= 1.0f ? 1.0f : c;  // NaN stays NaN
    }
}

// ------------------------------------------------------------ captured steps
constexpr int kCounters = 56;
struct Counters {
    gefenx_adamw_counter c[kCounters];
    int32_t n;
};
static_assert(sizeof(Counters) <= 4080, "kernel arguments");

// One thread a tensor: the step counter goes up by one, and its row gets what the host would have computed
// from it, in float64 as there.
__global__ __launch_bounds__(64) void k_adamw_counters(const Counters q) {
    const int i = threadIdx.x;
    if (i >= q.n) return;
    const gefenx_adamw_counter& c = q.c[i];
    const float t = *gbl(c.step) + 1.0f;
    *gbl(c.step) = t;
    const double lr = !c.lr_dev ? c.lr
                      : c.lr_dtype == GEFENX_F64 ? *gbl((const double*)c.lr_dev) : (double)*gbl((const float*)c.lr_dev);
    gefenx_adamw_row r;
    r.step_size = (float)(lr / (1.0 - pow(c.beta1, (double)t)));
    r.wd_factor = (float)(1.0 - lr * c.weight_decay);
    r.inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(c.beta2, (double)t)));
    r.reserved = 0;
    r.key = mix64(c.key0 + 0x9E3779B97F4A7C15ULL * (uint64_t)t);
    *c.row = r;
}

// ------------------------------------------------------------ host side
int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GEFENX_OK : set_error(GEFENX_ELAUNCH, "%s: %s", what, hipGetErrorString(e));
}

int validate(const char* what, const gefenx_adamw_desc* d, int n, bool state, bool param) {
    if (n < 0 || (n > 0 && !d)) return set_error(GEFENX_EINVAL, "%s: bad descriptor array (n=%d)", what, n);
    for (int i = 0; i < n; ++i) {
        if (d[i].dtype != GEFENX_F32 && d[i].dtype != GEFENX_F16 && d[i].dtype != GEFENX_BF16)
            return set_error(GEFENX_EDTYPE, "%s: tensor %d: unsupported dtype %d", what, i, d[i].dtype);
        if (d[i].bits != 8 && d[i].bits != 32)
            return set_error(GEFENX_EINVAL, "%s: tensor %d: moments of %d bits (8 or 32)", what, i, d[i].bits);
        if (d[i].numel < 0 || d[i].numel > kMaxNumel)
            return set_error(GEFENX_EINVAL, "%s: tensor %d: bad numel %lld", what, i, (long long)d[i].numel);
        if (d[i].numel == 0) continue;
        const bool scales = d[i].bits == 32 || (d[i].exp_avg_scale && d[i].exp_avg_sq_scale);
        if ((param && !d[i].p) || !d[i].grad || (state && (!d[i].exp_avg || !d[i].exp_avg_sq || !scales)))
            return set_error(GEFENX_EINVAL, "%s: tensor %d: null pointer", what, i);
    }
    return GEFENX_OK;
}

Item item_of(const gefenx_adamw_desc& d) {
    return Item{d.p, d.grad, d.exp_avg, d.exp_avg_sq, d.exp_avg_scale, d.exp_avg_sq_scale, d.numel, d.key,
                d.step_size, d.wd_factor, d.beta1, d.alpha1, d.beta2, d.alpha2, d.inv_sqrt_bc2, d.eps, d.row};
}

// Elements of a workgroup.  One pass each: workgroups start in order, so what is being written at any
// time lies in a few runs of memory (four passes: 960 us against 896 on the layer above).
constexpr int64_t kWg32 = (int64_t)kT * kW32, kWg8 = (int64_t)kT * kBlock8 / kGroup, kWgValues = (int64_t)kT * 4;
constexpr int64_t kNormPass = (int64_t)kT * 8;

// Calls launch(batch, workgroups) for the tensors that take(descriptor) picks, kItems at a time, `per`
// elements to a workgroup.
template <class P, class F>
int for_batches(const gefenx_adamw_desc* d, int n, int64_t per, P&& take, F&& launch) {
    Batch b;
    b.n = 0;
    b.iters = 1;
    int64_t wgs = 0;
    const auto flush = [&]() -> int {
        if (!b.n) return GEFENX_OK;
        const int rc = launch(b, (int)wgs);
        b.n = 0;
        wgs = 0;
        return rc;
    };
    for (int i = 0; i < n; ++i) {
        if (d[i].numel == 0 || !take(d[i])) continue;
        const int64_t w = (d[i].numel + per - 1) / per;
        if (b.n == kItems || wgs + w > kMaxWgs) {
            const int rc = flush();
            if (rc != GEFENX_OK) return rc;
        }
        b.it[b.n] = item_of(d[i]);
        wgs += w;
        b.end[b.n++] = (int32_t)wgs;
    }
    return flush();
}

int64_t total_elems(const gefenx_adamw_desc* d, int n) {
    int64_t s = 0;
    for (int i = 0; i < n; ++i) s += d[i].numel;
    return s;
}

int norm_iters(int64_t elems) {
    const int64_t k = (elems + kNormPartials * kNormPass - 1) / (kNormPartials * kNormPass);
    return (int)(k < 1 ? 1 : k);
}

int64_t norm_partials(const gefenx_adamw_desc* d, int n) {
    const int64_t per = kNormPass * norm_iters(total_elems(d, n));
    int64_t s = 0;
    for (int i = 0; i < n; ++i) s += (d[i].numel + per - 1) / per;
    return s;
}

// Whether eps is 2^24 times all that sqrt(v) / sqrt(bc2) can be for v < 2^-126.  bc2 = 1 - b2^t is
// 1 - b2 at least, so 2^-63 / sqrt(1 - b2) <= 2^-24 eps at every step (eps = 1e-8: b2 up to 1 - 3.3e-8).
bool drowns(float eps, float alpha2) { return (double)eps * eps * alpha2 >= 0x1p-78; }

template <int DT>
int step_dtype(const gefenx_adamw_desc* d, int n, const float* coef, hipStream_t s) {
    const auto picks = [](int bits, bool fast) {
        return [=](const gefenx_adamw_desc& t) {
            return t.dtype == DT && t.bits == bits && (bits == 32 || drowns(t.eps, t.alpha2) == fast);
        };
    };
    int rc = for_batches(d, n, kWg32, picks(32, false), [&](const Batch& b, int wgs) {
        k_adamw<DT><<<wgs, kT, 0, s>>>(b, coef);
        return launched("gefenx_adamw_step");
    });
    if (rc == GEFENX_OK)
        rc = for_batches(d, n, kWg8, picks(8, true), [&](const Batch& b, int wgs) {
            k_adamw8<DT, true><<<wgs, kT, 0, s>>>(b, coef);
            return launched("gefenx_adamw_step");
        });
    if (rc == GEFENX_OK)
        rc = for_batches(d, n, kWg8, picks(8, false), [&](const Batch& b, int wgs) {
            k_adamw8<DT, false><<<wgs, kT, 0, s>>>(b, coef);
            return launched("gefenx_adamw_step");
        });
    return rc;
}

template <int DT>
int norm_dtype(const gefenx_adamw_desc* d, int n, int iters, double*& at, hipStream_t s) {
    return for_batches(d, n, kNormPass * iters, [](const gefenx_adamw_desc& t) { return t.dtype == DT; }, [&](Batch& b, int wgs) {
        b.iters = iters;
        k_grad_sumsq<DT><<<wgs, kT, 0, s>>>(b, at);
        at += wgs;
        return launched("gefenx_adamw_norm");
    });
}

}  // namespace
}  // namespace gx

using namespace gx;

extern "C" {

int gefenx_adamw_step(const gefenx_adamw_desc* descs, int n, const float* grad_coef, void* stream) {
    int rc = validate("gefenx_adamw_step", descs, n, true, true);
    if (rc != GEFENX_OK) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    rc = step_dtype<F32>(descs, n, grad_coef, s);
    if (rc == GEFENX_OK) rc = step_dtype<F16>(descs, n, grad_coef, s);
    if (rc == GEFENX_OK) rc = step_dtype<BF16>(descs, n, grad_coef, s);
    return rc;
}

size_t gefenx_adamw_norm_workspace_bytes(const gefenx_adamw_desc* descs, int n) {
    if (validate("gefenx_adamw_norm_workspace_bytes", descs, n, false, false) != GEFENX_OK) return 0;
    return sizeof(double) * (size_t)(norm_partials(descs, n) + 1);
}

int gefenx_adamw_norm(const gefenx_adamw_desc* descs, int n, double max_norm, float* norm_out, void* workspace,
                      size_t workspace_bytes, void* stream) {
    int rc = validate("gefenx_adamw_norm", descs, n, false, false);
    if (rc != GEFENX_OK) return rc;
    if (!norm_out || !workspace || !(max_norm > 0.0))
        return set_error(GEFENX_EINVAL, "gefenx_adamw_norm: bad arguments (max_norm=%g)", max_norm);
    const int64_t partials = norm_partials(descs, n);
    if (workspace_bytes < sizeof(double) * (size_t)partials)
        return set_error(GEFENX_EINVAL, "gefenx_adamw_norm: workspace of %zu bytes, %zu needed", workspace_bytes,
                         sizeof(double) * (size_t)partials);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    double* at = static_cast<double*>(workspace);
    const int iters = norm_iters(total_elems(descs, n));
    rc = norm_dtype<F32>(descs, n, iters, at, s);
    if (rc == GEFENX_OK) rc = norm_dtype<F16>(descs, n, iters, at, s);
    if (rc == GEFENX_OK) rc = norm_dtype<BF16>(descs, n, iters, at, s);
    if (rc != GEFENX_OK) return rc;
    k_grad_norm<<<1, 1024, 0, s>>>(static_cast<const double*>(workspace), partials, max_norm, norm_out);
    return launched("gefenx_adamw_norm");
}

int gefenx_adamw_advance(const gefenx_adamw_counter* counters, int n, void* stream) {
    const char* what = "gefenx_adamw_advance";
    if (n < 0 || (n > 0 && !counters)) return set_error(GEFENX_EINVAL, "%s: bad array (n=%d)", what, n);
    for (int i = 0; i < n; ++i) {
        if (!counters[i].step || !counters[i].row) return set_error(GEFENX_EINVAL, "%s: tensor %d: null pointer", what, i);
        if (counters[i].lr_dev && counters[i].lr_dtype != GEFENX_F32 && counters[i].lr_dtype != GEFENX_F64)
            return set_error(GEFENX_EDTYPE, "%s: tensor %d: unsupported lr dtype %d", what, i, counters[i].lr_dtype);
    }
    for (int at = 0; at < n; at += kCounters) {
        Counters q;
        q.n = n - at < kCounters ? n - at : kCounters;
        for (int i = 0; i < q.n; ++i) q.c[i] = counters[at + i];
        k_adamw_counters<<<1, 64, 0, static_cast<hipStream_t>(stream)>>>(q);
        const int rc = launched(what);
        if (rc != GEFENX_OK) return rc;
    }
    return GEFENX_OK;
}

int gefenx_adamw_moments(const gefenx_adamw_desc* descs, int n, void* stream) {
    int rc = validate("gefenx_adamw_moments", descs, n, true, true);
    if (rc != GEFENX_OK) return rc;
    for (int i = 0; i < n; ++i)
        if (descs[i].bits != 8 || descs[i].dtype != GEFENX_F32)
            return set_error(GEFENX_EINVAL, "gefenx_adamw_moments: tensor %d: 8-bit moments into fp32 only", i);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return for_batches(descs, n, kWgValues, [](const gefenx_adamw_desc&) { return true; }, [&](const Batch& b, int wgs) {
        k_adamw8_values<<<wgs, kT, 0, s>>>(b);
        return launched("gefenx_adamw_moments");
    });
}

}  // extern "C"
