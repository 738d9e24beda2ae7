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

namespace gx {
namespace {

constexpr int kT = 256;                  // threads of a workgroup
constexpr int kItems = 36;               // tensors of a launch: 36 * 100 bytes of kernel arguments
constexpr int kBlock8 = 256;             // elements per scale of the 8-bit moments
constexpr int kGroup = 16;               // lanes that share such a block, two chunks of 8 elements each
constexpr float kTiny = 0x1p-126f;       // smallest scale: its reciprocal, and 448 of them, are finite
constexpr int kCode0 = 761;              // bits(x) >> 20 of v's code c is c + 761: code 255 is x = 1
constexpr int64_t kNormPartials = 4096;  // about so many partial sums of the gradient norm

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
};

struct Batch {
    Item it[kItems];
    int32_t end[kItems];  // workgroups up to and including tensor i
    int32_t n;
    int32_t iters;        // a workgroup's chunks per lane (8-bit moments: pairs of chunks)
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

// ------------------------------------------------------------ chunks of 8
// Whole chunks by vector accesses of any alignment, the last one of a tensor by elements.

template <int DT>
__device__ __forceinline__ void load_chunk(const typename Elem<DT>::T* base, int64_t left, Raw8<DT>& r) {
    if (left >= 8) {
        load_raw8_any<DT>(base, r);
        return;
    }
    if constexpr (DT == F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) r.f[k] = k < left ? *gbl(base + k) : 0.0f;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t lo = 2 * k < left ? *gbl(base + 2 * k) : 0, hi = 2 * k + 1 < left ? *gbl(base + 2 * k + 1) : 0;
            r.w[k] = lo | (hi << 16);
        }
    }
}

template <int DT>
__device__ __forceinline__ void store_chunk(typename Elem<DT>::T* base, int64_t left, const float v[8]) {
    if (left >= 8) {
        store8_any<DT>(base, v);
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k < left) *gbl(base + k) = from_f32<DT>(v[k]);
}

__device__ __forceinline__ RawIdx8 load_codes(const uint8_t* base, int64_t left) {
    if (left >= 8) return load_raw_idx8_any(base);
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k < left) w[k >> 2] |= (uint32_t)*gbl(base + k) << (8 * (k & 3));
    return RawIdx8{w[0], w[1]};
}

__device__ __forceinline__ void store_codes(uint8_t* base, int64_t left, const uint32_t w[2]) {
    if (left >= 8) {
        const u32x2 a = {w[0], w[1]};
        __builtin_nontemporal_store(a, GX_GLOBAL_AS(u32x2_a1, base));
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k < left) *gbl(base + k) = (uint8_t)(w[k >> 2] >> (8 * (k & 3)));
}

// The moments round after each operation, as the formula written in torch does, so 8-bit codes follow
// from the inputs alone.
__device__ __forceinline__ void advance(const Item& t, float g, float& m, float& v) {
    m = m * t.b1 + g * t.a1;
    v = v * t.b2 + g * g * t.a2;
}
__device__ __forceinline__ float stepped(const Item& t, float p, float m, float v) {
    const float d = __builtin_fmaf(__builtin_sqrtf(v), t.rbc2, t.eps);
    return __builtin_fmaf(-t.step, m / d, p * t.wdf);
}

// ------------------------------------------------------------ fp32 moments
template <int DT>
__global__ __launch_bounds__(kT) void k_adamw(const Batch b, const float* __restrict__ coef) {
    using T = typename Elem<DT>::T;
    int local;
    const Item& t = b.it[find_item(b, (int)blockIdx.x, local)];
    const float c = coef ? sload(coef) : 1.0f;
    for (int it = 0; it < b.iters; ++it) {
        const int64_t at = (((int64_t)local * b.iters + it) * kT + threadIdx.x) * 8;
        const int64_t left = t.n - at;
        if (left <= 0) return;
        Raw8<DT> g, p;
        Raw8<F32> m, v;
        load_chunk<DT>((const T*)t.g + at, left, g);
        load_chunk<F32>((const float*)t.m + at, left, m);
        load_chunk<F32>((const float*)t.v + at, left, v);
        load_chunk<DT>((const T*)t.p + at, left, p);
        float q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            advance(t, raw_elem<DT>(g, k) * c, m.f[k], v.f[k]);
            q[k] = stepped(t, raw_elem<DT>(p, k), m.f[k], v.f[k]);
        }
        store_chunk<F32>((float*)t.m + at, left, m.f);
        store_chunk<F32>((float*)t.v + at, left, v.f);
        store_chunk<DT>((T*)t.p + at, left, q);
    }
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

__device__ __forceinline__ void decode_m(const RawIdx8& c, float scale, float m[8]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.lo, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.lo, true);
    const f32x2 d = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.hi, false), e = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.hi, true);
    m[0] = a.x * scale; m[1] = a.y * scale; m[2] = b.x * scale; m[3] = b.y * scale;
    m[4] = d.x * scale; m[5] = d.y * scale; m[6] = e.x * scale; m[7] = e.y * scale;
}

__device__ __forceinline__ void decode_v(const RawIdx8& c, float scale, float v[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t x = raw_idx(c, k);
        v[k] = (x ? __uint_as_float((x + kCode0) << 20) : 0.0f) * scale;
    }
}

__device__ __forceinline__ void encode_m(const float m[8], float inv, uint32_t w[2]) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __builtin_amdgcn_fmed3f(m[k] * inv, -448.0f, 448.0f);
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], 0, false);
    w[0] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
    w[1] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], hi, true);
}

// at: the chunk's first element, a multiple of 8: two draws of four elements each
__device__ __forceinline__ void encode_v(const float v[8], float inv, uint64_t key, int64_t at, uint32_t w[2]) {
    constexpr uint64_t kGolden = 0x9E3779B97F4A7C15ULL;
    const uint64_t z0 = key + kGolden * ((uint64_t)(at >> 2) + 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint64_t z = mix64(h ? z0 + kGolden : z0);
        const uint32_t r[2] = {(uint32_t)z, (uint32_t)(z >> 32)};
        uint32_t packed = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t dither = (k & 1 ? r[k >> 1] >> 12 : r[k >> 1] << 4) & 0xffff0u;
            const float x = v[4 * h + k];
            int c = (int)((__float_as_uint(x * inv) + dither) >> 20) - kCode0;
            c = c < 1 ? 1 : (c > 255 ? 255 : c);
            packed |= (uint32_t)(x == 0.0f ? 0 : c) << (8 * k);
        }
        w[h] = packed;
    }
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

template <int DT>
__global__ __launch_bounds__(kT) void k_adamw8(const Batch b, const float* __restrict__ coef) {
    using T = typename Elem<DT>::T;
    int local;
    const Item& t = b.it[find_item(b, (int)blockIdx.x, local)];
    const float c = coef ? sload(coef) : 1.0f;
    const int lane = threadIdx.x & (kGroup - 1), group = threadIdx.x / kGroup;
    for (int it = 0; it < b.iters; ++it) {
        const int64_t blk = ((int64_t)local * b.iters + it) * (kT / kGroup) + group;
        const int64_t at0 = blk * kBlock8 + lane * 8;
        // the 16 lanes of a block leave together or stay together: what they exchange is among themselves
        if (blk * kBlock8 >= t.n) return;
        Raw8<DT> g[2], p[2];
        RawIdx8 mc[2], vc[2];
        const float ms = *gbl(t.ms + blk), vs = *gbl(t.vs + blk);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t at = at0 + h * (kBlock8 / 2), left = t.n - at;
            load_chunk<DT>((const T*)t.g + at, left, g[h]);
            mc[h] = load_codes((const uint8_t*)t.m + at, left);
            vc[h] = load_codes((const uint8_t*)t.v + at, left);
            load_chunk<DT>((const T*)t.p + at, left, p[h]);
        }
        float m[2][8], v[2][8];
        uint32_t mx = 0, vx = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t at = at0 + h * (kBlock8 / 2), left = t.n - at;
            decode_m(mc[h], ms, m[h]);
            decode_v(vc[h], vs, v[h]);
            float q[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                advance(t, raw_elem<DT>(g[h], k) * c, m[h][k], v[h][k]);
                q[k] = stepped(t, raw_elem<DT>(p[h], k), m[h][k], v[h][k]);
                const uint32_t mb = __float_as_uint(m[h][k]) & 0x7fffffffu, vb = __float_as_uint(v[h][k]) & 0x7fffffffu;
                mx = mb > mx ? mb : mx;
                vx = vb > vx ? vb : vx;
            }
            if (left > 0) store_chunk<DT>((T*)t.p + at, left, q);
        }
        const float mscale = block_scale(__uint_as_float(group16_max(mx)) * (1.0f / 448.0f));
        const float vscale = block_scale(__uint_as_float(group16_max(vx)));
        const float minv = 1.0f / mscale, vinv = 1.0f / vscale;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t at = at0 + h * (kBlock8 / 2), left = t.n - at;
            uint32_t w[2];
            encode_m(m[h], minv, w);
            if (left > 0) store_codes((uint8_t*)t.m + at, left, w);
            encode_v(v[h], vinv, t.key, at, w);
            if (left > 0) store_codes((uint8_t*)t.v + at, left, w);
        }
        if (lane == 0) {
            *gbl(t.ms + blk) = mscale;
            *gbl(t.vs + blk) = vscale;
        }
    }
}

// The values that 8-bit moments stand for: Item::p and Item::g are where m's and v's go.
__global__ __launch_bounds__(kT) void k_adamw8_values(const Batch b) {
    int local;
    const Item& t = b.it[find_item(b, (int)blockIdx.x, local)];
    for (int it = 0; it < b.iters; ++it) {
        const int64_t at = (((int64_t)local * b.iters + it) * kT + threadIdx.x) * 8;
        const int64_t left = t.n - at;
        if (left <= 0) return;
        const RawIdx8 mc = load_codes((const uint8_t*)t.m + at, left), vc = load_codes((const uint8_t*)t.v + at, left);
        const int64_t blk = at / kBlock8;
        float x[8];
        decode_m(mc, *gbl(t.ms + blk), x);
        store_chunk<F32>((float*)t.p + at, left, x);
        decode_v(vc, *gbl(t.vs + blk), x);
        store_chunk<F32>((float*)const_cast<void*>(t.g) + at, left, x);
    }
}

// ------------------------------------------------------------ gradient norm
// Sums of squares in float64, one partial per workgroup, added up by one workgroup in a fixed order.
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
        Raw8<DT> g;
        load_chunk<DT>((const T*)t.g + at, left, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const double x = (double)raw_elem<DT>(g, k);
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
        if (d[i].numel < 0 || d[i].numel >= (int64_t)1 << 40)
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
                d.step_size, d.wd_factor, d.beta1, d.alpha1, d.beta2, d.alpha2, d.inv_sqrt_bc2, d.eps};
}

// Elements of one pass of a workgroup.
constexpr int64_t kPass32 = (int64_t)kT * 8, kPass8 = (int64_t)kT * 16;

// Calls launch(batch, workgroups) for the tensors of one dtype and moment width, kItems at a time.
template <class F>
int for_batches(const gefenx_adamw_desc* d, int n, int dtype, int bits, int64_t pass, int iters, F&& launch) {
    Batch b;
    b.n = 0;
    b.iters = iters;
    int64_t wgs = 0;
    const auto flush = [&]() -> int {
        if (!b.n) return GEFENX_OK;
        const int rc = launch(b, (int)wgs);
        b.n = 0;
        wgs = 0;
        return rc;
    };
    for (int i = 0; i < n; ++i) {
        if (d[i].dtype != dtype || (bits && d[i].bits != bits) || d[i].numel == 0) continue;
        const int64_t w = (d[i].numel + pass * iters - 1) / (pass * iters);
        if (b.n == kItems || wgs + w > 0x3fffffff) {
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

int step_iters(int64_t elems, int64_t pass) {
    return elems >= (int64_t)8192 * pass ? 4 : 1;
}

int norm_iters(int64_t elems) {
    const int64_t k = (elems + kNormPartials * kPass32 - 1) / (kNormPartials * kPass32);
    return (int)(k < 1 ? 1 : k);
}

int64_t norm_partials(const gefenx_adamw_desc* d, int n) {
    const int64_t per = kPass32 * norm_iters(total_elems(d, n));
    int64_t s = 0;
    for (int i = 0; i < n; ++i) s += (d[i].numel + per - 1) / per;
    return s;
}

template <int DT>
int step_dtype(const gefenx_adamw_desc* d, int n, int64_t elems, const float* coef, hipStream_t s) {
    int rc = for_batches(d, n, DT, 32, kPass32, step_iters(elems, kPass32), [&](const Batch& b, int wgs) {
        k_adamw<DT><<<wgs, kT, 0, s>>>(b, coef);
        return launched("gefenx_adamw_step");
    });
    if (rc != GEFENX_OK) return rc;
    return for_batches(d, n, DT, 8, kPass8, step_iters(elems, kPass8), [&](const Batch& b, int wgs) {
        k_adamw8<DT><<<wgs, kT, 0, s>>>(b, coef);
        return launched("gefenx_adamw_step");
    });
}

template <int DT>
int norm_dtype(const gefenx_adamw_desc* d, int n, int iters, double*& at, hipStream_t s) {
    return for_batches(d, n, DT, 0, kPass32, iters, [&](const Batch& b, int wgs) {
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
    const int64_t elems = total_elems(descs, n);
    rc = step_dtype<F32>(descs, n, elems, grad_coef, s);
    if (rc == GEFENX_OK) rc = step_dtype<F16>(descs, n, elems, grad_coef, s);
    if (rc == GEFENX_OK) rc = step_dtype<BF16>(descs, n, elems, grad_coef, s);
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

int gefenx_adamw_moments(const gefenx_adamw_desc* descs, int n, void* stream) {
    int rc = validate("gefenx_adamw_moments", descs, n, true, true);
    if (rc != GEFENX_OK) return rc;
    for (int i = 0; i < n; ++i)
        if (descs[i].bits != 8 || descs[i].dtype != GEFENX_F32)
            return set_error(GEFENX_EINVAL, "gefenx_adamw_moments: tensor %d: 8-bit moments into fp32 only", i);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return for_batches(descs, n, F32, 8, kPass32, step_iters(total_elems(descs, n), kPass32), [&](const Batch& b, int wgs) {
        k_adamw8_values<<<wgs, kT, 0, s>>>(b);
        return launched("gefenx_adamw_moments");
    });
}

}  // extern "C"
