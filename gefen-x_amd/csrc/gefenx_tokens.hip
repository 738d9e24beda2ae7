// gefenx_tokens.hip -- statistics of tokens over the logits of a language model, and distillation from a teacher's
// likeliest tokens, with the gradients of the logits.
//
// With z = x / tau, m = max z, S = sum exp(z - m), T = sum (z - m) exp(z - m), q = exp(z - m) / S:
//   statistics:   log q[y];  entropy H = log S - T / S;  the largest x, ties by the lowest index
//     d / d z_v = [v = y] g + sum_j [v = i_j] g_j - q_v (g + sum_j g_j + g_H (log q_v + H))
//   distillation: D = sum_j p_j (log p_j - log q[i_j]), and for the others r (log r - log rho) with
//     r = 1 - sum p, rho = 1 - sum q[i_j] = R / S, R the sum over the logits outside of the teacher's tokens
//     d D / d z_v = (P + r) q_v - p_v for the teacher's tokens, q_v (P + r - r / rho) elsewhere
//     loss = mean over rows of (1 - w) tau^2 D - w log softmax(x)[y]
// A pass over the logits for the sums, a few numbers per row, and a pass that writes the gradient.
#include "gefenx_hunt.h"
#include "gefenx_logits.h"

namespace gx {
namespace {

constexpr int64_t kCus = 256;
constexpr int kMaxTop = 128;      // likeliest tokens of a row
constexpr int kMaxTeacher = 512;  // a teacher's tokens of a row
constexpr int kMergeKeys = 2048;  // candidates of a row's splits that are merged
constexpr int kBits = 16384;      // runs of a workgroup's part of a row where some are marked
// Differences from the maximum stop here: exp is 0 from there at any temperature, and 0 times it is 0.
constexpr float kFar = -1e25f;

// exp(d / tau) = 2^(d (hi + lo)), hi + lo = log2(e) / tau.  lo > 0: -inf times either is -inf.  inv_hi: 1 / hi; tilt:
// (hi / (hi + lo) - 1) / tau.
struct Heat {
    float hi, lo, inv, inv_hi, tilt;
    double inv64;
};
__device__ __forceinline__ float heat_exp(float d, const Heat& h) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, h.lo, d * h.hi));
}

// A running maximum m of x and s = sum exp((x - m) / tau); u: sum of (x - m) exp((x - m) / tau), or of exp(x - m).
// The maximum of nothing is -inf, and -inf logits add 0; NaN and +inf logits make the sums NaN.
enum { kNone = 0, kEntropy = 1, kPlain = 2 };
template <int U> struct Sums {
    float m = -__builtin_inff(), s = 0.0f, u = 0.0f;
    __device__ __forceinline__ void rebase(float m2, const Heat& h) {
        if (m2 > m) {
            const float d = m - m2, f = heat_exp(d, h);
            if (U == kEntropy) u = f * __builtin_fmaf(s, __builtin_fmaxf(d, kFar), u);
            if (U == kPlain) u = u * exp_(d);
            s = s * f;
            m = m2;
        }
    }
    __device__ __forceinline__ float base() const { return m == -__builtin_inff() ? 0.0f : m; }
    __device__ __forceinline__ void add(float x, float b, const Heat& h) {
        const float d = x - b, e = heat_exp(d, h);
        s += e;
        if (U == kEntropy) u = __builtin_fmaf(__builtin_fmaxf(d, kFar), e, u);
        if (U == kPlain) u += exp_(d);
    }
    __device__ __forceinline__ void join(float m2, float s2, float u2, const Heat& h) {
        const float top = m2 > m ? m2 : m;
        const float b = top == -__builtin_inff() ? 0.0f : top;
        const float da = m - b, db = m2 - b, fa = heat_exp(da, h), fb = heat_exp(db, h);
        if (U == kEntropy)
            u = fa * __builtin_fmaf(s, __builtin_fmaxf(da, kFar), u) + fb * __builtin_fmaf(s2, __builtin_fmaxf(db, kFar), u2);
        if (U == kPlain) u = u * exp_(da) + u2 * exp_(db);
        s = s * fa + s2 * fb;
        m = top;
    }
};

// The sums of a group of lanes, in every one of them: to their maximum first, then plain sums.
template <int U>
__device__ __forceinline__ void wave_join(Sums<U>& a, const Heat& h, int lanes = 64) {
    float top = a.m;
    for (int off = lanes >> 1; off > 0; off >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, off, 64));
    const float d = a.m - (top == -__builtin_inff() ? 0.0f : top), f = heat_exp(d, h);
    if (U == kEntropy) a.u = f * __builtin_fmaf(a.s, __builtin_fmaxf(d, kFar), a.u);
    if (U == kPlain) a.u *= exp_(d);
    a.s *= f;
    a.m = top;
    for (int off = lanes >> 1; off > 0; off >>= 1) {
        a.s += __shfl_xor(a.s, off, 64);
        if (U != kNone) a.u += __shfl_xor(a.u, off, 64);
    }
}

template <int U, int TH = kT>
__device__ __forceinline__ Sums<U> group_join(Sums<U> a, const Heat& h, float4* waves) {
    wave_join(a, h);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = make_float4(a.m, a.s, a.u, 0.0f);
    __syncthreads();
    a.m = waves[0].x;
    a.s = waves[0].y;
    a.u = waves[0].z;
#pragma unroll
    for (int w = 1; w < TH / 64; ++w) a.join(waves[w].x, waves[w].y, waves[w].z, h);
    return a;
}

// Sums as a lane takes them over its logits: 2^(x hi - M) with M = m hi rounded is one fused operation where
// 2^((x - m) (hi + lo)) is three (the statistics of 4096 x 128256 bf16 are bound by such operations as much as by
// memory).  What M's rounding and hi's make of the sums is known and put right in sums(): 2^(m hi - M) for all of
// them, and by hi alone s grows by (hi / (hi + lo) - 1) sum z exp(z), which u gives; without u the product with lo is
// taken too.  Where M is beyond kHuge its rounding would be more than half a power of two, or x hi overflow (rows that
// a mask of -1e10 or the type's lowest value leaves nothing): there the difference is taken first, and a maximum that
// passes kHuge takes what the lane has so far from one scale to the other.
constexpr float kHuge = 16777216.0f;
template <int U> struct LaneSums {
    float m = -__builtin_inff(), s = 0.0f, u = 0.0f, minus = 0.0f, minus1 = 0.0f;  // -M, and that of exp(x)
    static __device__ __forceinline__ bool huge(float of, float of1) {
        return __builtin_fabsf(of) > kHuge || (U == kPlain && __builtin_fabsf(of1) > kHuge);
    }
    __device__ __forceinline__ bool huge() const { return huge(minus, minus1); }
    // the exponents that a term of x = m has in s, and in kPlain's u: what the roundings leave of 0
    static __device__ __forceinline__ void offsets(float m, float of, float of1, const Heat& h, float& off, float& off1) {
        off = off1 = 0.0f;
        if (huge(of, of1)) return;
        off = __builtin_fmaf(m, h.hi, of);
        if (U != kEntropy) off = __builtin_fmaf(m, h.lo, off);
        off1 = __builtin_fmaf(m, kLog2eRest, __builtin_fmaf(m, kLog2e, of1));
    }
    __device__ __forceinline__ void rebase(float m2, const Heat& h) {
        if (!(m2 > m)) return;
        const float next = -(m2 * h.hi), next1 = -(m2 * kLog2e);
        if (m != -__builtin_inff()) {
            float d = next - minus, d1 = next1 - minus1;
            if (huge() || huge(next, next1)) {
                const float by = m - m2;
                float from, from1, to, to1;
                offsets(m, minus, minus1, h, from, from1);
                offsets(m2, next, next1, h, to, to1);
                d = (U == kEntropy ? by * h.hi : __builtin_fmaf(by, h.lo, by * h.hi)) + (to - from);
                d1 = __builtin_fmaf(by, kLog2eRest, by * kLog2e) + (to1 - from1);
            }
            const float f = __builtin_amdgcn_exp2f(d);
            if (U == kEntropy) u = f * __builtin_fmaf(s, __builtin_fmaxf(d, kFar), u);
            if (U == kPlain) u *= __builtin_amdgcn_exp2f(d1);
            s *= f;
        }
        m = m2;
        minus = next;
        minus1 = next1;
    }
    // FAR: y may be -inf, whose exponential of 0 times it would be NaN
    template <bool FAR> __device__ __forceinline__ void exponent(float y) {
        const float e = __builtin_amdgcn_exp2f(y);
        s += e;
        if (U == kEntropy) u = __builtin_fmaf(FAR ? __builtin_fmaxf(y, kFar) : y, e, u);
    }
    template <bool FAR> __device__ __forceinline__ void add(float x, const Heat& h) {
        const float y = __builtin_fmaf(x, h.hi, minus);
        exponent<FAR>(U == kEntropy ? y : __builtin_fmaf(x, h.lo, y));
        if (U == kPlain) u += __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2eRest, __builtin_fmaf(x, kLog2e, minus1)));
    }
    __device__ __forceinline__ void add_far(float x, const Heat& h) {
        const float d = x - m;
        exponent<true>(U == kEntropy ? d * h.hi : __builtin_fmaf(d, h.lo, d * h.hi));
        if (U == kPlain) u += exp_(d);
    }
    __device__ __forceinline__ Sums<U> sums(const Heat& h) const {
        Sums<U> a;
        a.m = m;
        float off = 0.0f, off1 = 0.0f;
        if (m != -__builtin_inff()) offsets(m, minus, minus1, h, off, off1);
        const float f = __builtin_amdgcn_exp2f(-off);
        a.s = s * f;
        if (U == kEntropy) {
            a.u = __builtin_fmaf(-off, s, u) * f * h.inv_hi;
            a.s = __builtin_fmaf(-h.tilt, a.u, a.s);
        }
        if (U == kPlain) a.u = u * __builtin_amdgcn_exp2f(-off1);
        return a;
    }
};

// The largest of N runs; fp16 goes two at a time.
template <int DT, int N>
__device__ __forceinline__ float largest(const Run<typename Elem<DT>::T, kW<DT>>* r) {
    if constexpr (DT == F16) {
        typedef _Float16 H2 __attribute__((ext_vector_type(2)));
        H2 top = {-__builtin_inff16(), -__builtin_inff16()};
#pragma unroll
        for (int c = 0; c < N; ++c) {
            H2 v[kW<DT> / 2];
            __builtin_memcpy(v, &r[c], sizeof(v));
#pragma unroll
            for (int k = 0; k < kW<DT> / 2; ++k) top = __builtin_elementwise_max(top, v[k]);
        }
        return __builtin_fmaxf((float)top.x, (float)top.y);
    } else {
        float top = -__builtin_inff();
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int k = 0; k < kW<DT>; ++k) top = __builtin_fmaxf(top, to_f32<DT>(r[c].e[k]));
        return top;
    }
}

// Adds N runs, the largest of which is top.
template <int DT, int U, int N>
__device__ __forceinline__ void add_runs(LaneSums<U>& a, const Run<typename Elem<DT>::T, kW<DT>>* r, float top, const Heat& h) {
    a.rebase(top, h);
    const float s = a.s, u = a.u;  // N runs are added up by themselves: a long row's sum keeps more of them
    a.s = a.u = 0.0f;
    if (!a.huge()) {
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int k = 0; k < kW<DT>; ++k) a.template add<false>(to_f32<DT>(r[c].e[k]), h);
    }
    if (a.huge() || (U == kEntropy && a.u != a.u && a.s == a.s)) {  // again: among them were huge ones, or -inf
        a.s = a.u = 0.0f;
#pragma unroll
        for (int c = 0; c < N; ++c) {
            // from the words anew: values kept for here would cost the pass its registers
            u32x4 words;
            __builtin_memcpy(&words, &r[c], sizeof(words));
            asm volatile("" : "+v"(words));
            Run<typename Elem<DT>::T, kW<DT>> v;
            __builtin_memcpy(&v, &words, sizeof(v));
#pragma unroll
            for (int k = 0; k < kW<DT>; ++k) {
                const float x = to_f32<DT>(v.e[k]);
                if (a.huge()) a.add_far(x, h);
                else a.template add<true>(x, h);
            }
        }
    }
    a.s += s;
    a.u += u;
}

// Runs begin .. end - 1 of a row, TH lanes at a time in steps of kStep runs each; each lane's sums.  skip(run): a
// run that is left out; note(a, b): the largest of the first and of the second half of a lane's step.  Which logits a
// lane adds up does not depend on where the row starts in memory.
template <int DT, int U, int TH, bool STREAM, class Skip, class Note>
__device__ __forceinline__ Sums<U> row_sums(const typename Elem<DT>::T* x, int64_t vocab, int64_t begin, int64_t end, int lane,
                                            const Heat& h, Skip&& skip, Note&& note) {
    using T = typename Elem<DT>::T;
    constexpr int W = kW<DT>;
    const int64_t whole = end * W <= vocab ? end : end - 1;
    const int64_t last = end * W < vocab ? end * W : vocab;  // column behind the part
    LaneSums<U> a;
    int64_t c = begin;
    const auto put = [&](Run<T, W>& v, int64_t run) {
        if (skip(run)) {
#pragma unroll
            for (int k = 0; k < W; ++k) v.e[k] = DT == F32 ? (T)-__builtin_inff() : (T)(DT == BF16 ? 0xff80 : 0xfc00);
        }
    };
    const auto add = [&](auto load) {
        for (; c + kStep * TH <= whole; c += kStep * TH) {
            Run<T, W> v[kStep];
#pragma unroll
            for (int i = 0; i < kStep; ++i) v[i] = load(x + (c + lane + i * TH) * W);
#pragma unroll
            for (int i = 0; i < kStep; ++i) put(v[i], c + lane + i * TH);
            const float one = largest<DT, kStep / 2>(v), two = largest<DT, kStep / 2>(v + kStep / 2);
            add_runs<DT, U, kStep>(a, v, __builtin_fmaxf(one, two), h);
            note(one, two);
        }
    };
    if (DT != F32 && ((uintptr_t)x & 3)) add([](const T* p) { return load_odd<DT, STREAM>(p); });
    else add([](const T* p) { return load_logits<DT, STREAM>(p); });
    if (c < end) {  // the last step, of which some runs are missing or not whole
        Run<T, W> v[kStep];
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
            const int64_t at = (c + lane + i * TH) * W;
            v[i] = load_logits<DT, STREAM>(x + at, last - at);
        }
        float half[2] = {-__builtin_inff(), -__builtin_inff()};
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
            if (c + i * TH >= end) break;
            if (c + lane + i * TH < end) put(v[i], c + lane + i * TH);
            const float top = largest<DT, 1>(v + i);
            add_runs<DT, U, 1>(a, v + i, top, h);
            half[i / (kStep / 2)] = __builtin_fmaxf(half[i / (kStep / 2)], top);
        }
        note(half[0], half[1]);
    }
    return a.sums(h);
}

// ------------------------------------------------------------ the likeliest tokens
// Logits in the order of their values as whole numbers above 0, NaN above all; -0 is 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    x += 0.0f;
    const uint32_t b = __float_as_uint(x);
    if (x != x) return 0xffffffffu;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
    if (o == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// Order and column as one number: of equal logits the lower column is the larger.  0 is no logit.
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t column) { return (uint64_t)order << 32 | (uint32_t)~column; }

// A barrier of a group of lanes: a workgroup, or a wave of it.
template <int TH> __device__ __forceinline__ void meet() {
    if constexpr (TH == kT) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

template <int TH> struct Select {
    uint32_t bins[256];
    uint32_t count, digit, above;
    uint32_t waves[TH / 64];
};

// The first `want` columns of first .. last - 1 whose order is `order`, as keys; waves: of TH / 64.
template <int DT, int TH>
__device__ __forceinline__ void first_equal(const typename Elem<DT>::T* x, int64_t first, int64_t last, uint32_t order,
                                            uint32_t want, uint32_t* waves, uint64_t* __restrict__ out) {
    const int lane = threadIdx.x % TH;
    uint32_t taken = 0;
    for (int64_t begin = first; taken < want && begin < last; begin += TH) {
        const int64_t v = begin + lane;
        const bool equal = v < last && order_of(to_f32<DT>(*gbl(x + v))) == order;
        const uint64_t who = __ballot(equal);
        uint32_t before = taken + (uint32_t)__popcll(who & (((uint64_t)1 << (lane & 63)) - 1));
        if constexpr (TH == 64) {
            taken += (uint32_t)__popcll(who);
        } else {
            __syncthreads();
            if ((lane & 63) == 0) waves[lane >> 6] = (uint32_t)__popcll(who);
            __syncthreads();
            for (int w = 0; w < TH / 64; ++w) {
                if (w < lane >> 6) before += waves[w];
                taken += waves[w];
            }
        }
        if (equal && before < want) out[before] = key_of(order, (uint32_t)v);
    }
}

// The `top` largest keys of columns first .. last - 1 of a row, in no order, 0 behind them, by digits of 8 bits of
// the order from the highest: after the last one the order of the top-th largest is known, larger ones are taken as
// they come, equal ones by column.
template <int DT, int TH>
__device__ __forceinline__ void select_keys(const typename Elem<DT>::T* x, int64_t first, int64_t last, int top, Select<TH>& at,
                                            uint64_t* __restrict__ out) {
    const int lane = threadIdx.x % TH;
    const auto order = [&](int64_t v) { return order_of(to_f32<DT>(*gbl(x + v))); };
    if (last - first <= top) {
        for (int64_t i = lane; i < top; i += TH) out[i] = first + i < last ? key_of(order(first + i), (uint32_t)(first + i)) : 0;
        return;
    }
    uint32_t prefix = 0, mask = 0, want = (uint32_t)top;
    for (int shift = 24; shift >= 0; shift -= 8) {
        meet<TH>();
        for (int i = lane; i < 256; i += TH) at.bins[i] = 0;
        at.count = 0;
        meet<TH>();
        for (int64_t v = first + lane; v < last; v += TH) {
            const uint32_t o = order(v);
            if ((o & mask) == prefix) atomicAdd(&at.bins[o >> shift & 255], 1u);
        }
        meet<TH>();
        if (lane == 0) {
            uint32_t above = 0, d = 255;
            while (d > 0 && above + at.bins[d] < want) above += at.bins[d--];
            at.digit = d;
            at.above = above;
        }
        meet<TH>();
        want -= at.above;
        prefix |= at.digit << shift;
        mask |= 255u << shift;
    }
    for (int64_t v = first + lane; v < last; v += TH) {
        const uint32_t o = order(v);
        if (o > prefix) out[atomicAdd(&at.count, 1u)] = key_of(o, (uint32_t)v);
    }
    first_equal<DT, TH>(x, first, last, prefix, want, at.waves, out + (top - want));
}

// The want-th largest (want <= TH) of the orders that a group's lanes bring, or 0, by bits from the highest that the
// type's values tell apart.  A workgroup's first wave looks through all of them, four to a lane, the others wait.
template <int DT, int TH>
__device__ __forceinline__ uint32_t largest_of_lanes(uint32_t own, int want, uint32_t* all) {
    constexpr int kLast = DT == F32 ? 0 : DT == F16 ? 13 : 16, N = TH / 64;
    uint32_t v[N] = {own}, found = 0;
    if constexpr (N > 1) {
        all[threadIdx.x] = own;
        __syncthreads();
    }
    if (N == 1 || threadIdx.x < 64) {
        if constexpr (N > 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = all[i * 64 + threadIdx.x];
        }
#pragma unroll 4
        for (int bit = 31; bit >= kLast; --bit) {
            const uint32_t next = found | 1u << bit;
            int n = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) n += (int)__popcll(__ballot(v[i] >= next));
            if (n >= want) found = next;
        }
    }
    if constexpr (N > 1) {
        if (threadIdx.x == 0) all[0] = found;
        __syncthreads();
        found = all[0];
    }
    // below, a value's order has zeros where it is positive and ones where it is negative
    return found | (found >> 31 || found == 0 ? 0 : (1u << kLast) - 1);
}

// What the rows come to.
struct Statistics {
    float *logps, *entropy, *top_logps;
    int64_t* top_ids;
    float4* stats;  // {maximum, sum, log of the sum, entropy}
};

__device__ __forceinline__ void ignored_row(const Statistics& out, int64_t r, int top, int lane, int lanes) {
    if (lane == 0) {
        if (out.logps) out.logps[r] = 0.0f;
        out.entropy[r] = 0.0f;
        out.stats[r] = make_float4(0.0f, 1.0f, 0.0f, 0.0f);
    }
    for (int i = lane; i < top; i += lanes) {
        out.top_ids[r * top + i] = 0;
        out.top_logps[r * top + i] = -__builtin_inff();
    }
}

template <int DT>
__device__ __forceinline__ float label_logit(const Rows& q, const typename Elem<DT>::T* x, int64_t label) {
    return q.labels && (uint64_t)label < (uint64_t)q.vocab ? to_f32<DT>(*gbl(x + label)) : 0.0f;
}

// A row's maximum and the log of its sum: a log-probability is (x - max) / tau - log_sum.
struct Level {
    double max, log_sum;
};

// A row's sums and its label's logit x to its results, by one lane.
__device__ __forceinline__ Level row_results(const Rows& q, const Heat& h, const Statistics& out, int64_t r, int64_t label,
                                              float x, const Sums<kEntropy>& a) {
    const double log_sum = log((double)a.s);
    const float entropy = (float)(log_sum - (double)a.u / (double)a.s * h.inv64);
    if (out.logps)
        out.logps[r] = (uint64_t)label < (uint64_t)q.vocab ? (float)(((double)x - (double)a.m) * h.inv64 - log_sum)
                                                           : __uint_as_float(0x7fc00000u);
    out.entropy[r] = entropy;
    out.stats[r] = make_float4(a.m, a.s, (float)log_sum, entropy);
    return {(double)a.m, log_sum};
}

__device__ __forceinline__ void top_result(const Heat& h, const Statistics& out, int64_t at, uint64_t key, const Level& level) {
    out.top_ids[at] = (int64_t)(uint32_t)~(uint32_t)key;
    out.top_logps[at] = (float)(((double)value_of((uint32_t)(key >> 32)) - level.max) * h.inv64 - level.log_sum);
}

// The place of each of n keys (no two alike) among them: put(place, key) for the `top` largest.  keys: at a multiple of
// 16 bytes, and room for one more.
template <int TH, class Put>
__device__ __forceinline__ void by_rank(uint64_t* keys, int n, int top, Put&& put) {
    if (threadIdx.x % TH == 0) keys[n] = 0;
    meet<TH>();
    const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(keys);
    for (int i = threadIdx.x % TH; i < n; i += TH) {
        const uint64_t key = keys[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; j += 2) {
            const ulonglong2 two = pairs[j / 2];
            rank += (two.x > key ? 1 : 0) + (two.y > key ? 1 : 0);
        }
        if (rank < top) put(rank, key);
    }
}

// The maxima of both halves of a lane's step in a word: of 2-byte logits each, of fp32 ones the larger.
template <int DT> struct Maxima {
    static constexpr int kParts = DT == F32 ? 1 : 2;
    static __device__ __forceinline__ uint32_t put(float a, float b) {
        if constexpr (DT == F32) return __float_as_uint(__builtin_fmaxf(a, b));
        else return (uint32_t)from_f32<DT>(a) | (uint32_t)from_f32<DT>(b) << 16;
    }
    static __device__ __forceinline__ float get(uint32_t w, int part) {
        if constexpr (DT == F32) return __uint_as_float(w);
        else return to_f32<DT>((uint16_t)(w >> 16 * part));
    }
};

// Maxima of a lane of a wave that has a row of its own; how many maxima are looked through again.
constexpr int kWaveSlots = (int)kShortRuns / (64 * kStep);
constexpr int kWaveTop = 32;  // likeliest tokens that a wave finds for a row of its own
template <int TH> constexpr int kSuspects = TH == kT ? 384 : 128;
template <int TH> struct Hunt {
    uint16_t suspects[kSuspects<TH>];
    uint32_t n_suspects, n_candidates, waves[TH / 64];
    Level level;
};

// part[row][split] = the sums of a split of a row, keys[row][split][top] its largest, 0 where there are fewer; a whole
// row's results at once.  PER rows to a workgroup: one, or one for each of its waves (rows without splits).
//
// The likeliest tokens cost the pass a maximum of each step of a lane, kept in LDS.  The top-th largest of the lanes'
// maxima is a bound that at least `top` logits reach; the few steps that reach it are read again, what reaches it in
// them are the candidates, and counting the larger ones gives each its place.  More candidates than there is room for
// (equal logits) are those over the bound and the first of the equal ones; NaN, +inf and what is left go through
// select_keys.
//
// 4096 x 128256 bf16: 163-175 us, 6.0-6.4 TB/s, the vector units busy 79% of it (7.2 instructions a logit: convert,
// the maximum, fma, exp, the two sums); with 64 tokens 186 us, 7% read again for them.  16384 x 1000 fp32 14 us.
template <int DT, int PER, bool TOP>
__global__ __launch_bounds__(kT) void k_statistics(const Rows q, const Heat h, int top, int steps_of_slot, int room, const Statistics out,
                                                   float4* __restrict__ part, uint64_t* __restrict__ keys) {
    using T = typename Elem<DT>::T;
    constexpr int TH = kT / PER, W = kW<DT>;
    __shared__ float4 waves[kT / 64];
    __shared__ std::conditional_t<TOP, Hunt<TH>, char> hunts[PER];
    extern __shared__ __align__(16) uint64_t dynamic[];
    const int lane = threadIdx.x % TH, wave = PER > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TH) : 0;
    const int64_t at = (int64_t)blockIdx.x * PER + wave;
    const int64_t r = PER > 1 ? at : at / (uint32_t)q.splits, split = PER > 1 ? 0 : at % (uint32_t)q.splits;
    if (r >= q.rows) return;
    const int64_t label = q.labels ? sload(q.labels + r) : 0;
    const bool alone = PER > 1 || q.splits == 1;
    if (q.labels && label == q.ignore) {
        if (alone) ignored_row(out, r, top, lane, TH);
        return;
    }
    const int64_t runs = (q.vocab + W - 1) / W, begin = split * q.split_runs;
    const int64_t end = begin + q.split_runs < runs ? begin + q.split_runs : runs;
    const T* x = (const T*)q.x + row_offset(q, r);
    const float xl = alone ? label_logit<DT>(q, x, label) : 0.0f;  // on its way early
    const auto none = [](int64_t) { return false; };
    const int slots = TOP && begin < end ? slots_of(end - begin, TH, steps_of_slot) : 0;  // no more than a whole split's
    uint64_t* own_lds = dynamic + (PER > 1 ? wave * hunt_words(TH, kWaveSlots) : 0);
    uint32_t* tops = reinterpret_cast<uint32_t*>(own_lds);
    uint32_t* slot = tops + lane;
    float held[2] = {-__builtin_inff(), -__builtin_inff()};
    int to_go = steps_of_slot;
    const auto note = [&](float one, float two) {
        if constexpr (TOP) {
            held[0] = __builtin_fmaxf(held[0], one);
            held[1] = __builtin_fmaxf(held[1], two);
            *slot = Maxima<DT>::put(held[0], held[1]);
            if (--to_go == 0) {
                to_go = steps_of_slot;
                held[0] = held[1] = -__builtin_inff();
                slot += TH;
            }
        }
    };
    Sums<kEntropy> a = q.cached ? row_sums<DT, kEntropy, TH, false>(x, q.vocab, begin, end, lane, h, none, note)
                                : row_sums<DT, kEntropy, TH, true>(x, q.vocab, begin, end, lane, h, none, note);
    const float own = a.m;
    if constexpr (PER > 1) wave_join(a, h);
    else a = group_join(a, h, waves);
    if constexpr (!TOP) {
        if (lane == 0) {
            if (alone) row_results(q, h, out, r, label, xl, a);
            else part[at] = make_float4(a.m, a.s, a.u, 0.0f);
        }
    } else {
        Hunt<TH>& hunt = hunts[wave];
        if (lane == 0) {
            hunt.n_suspects = hunt.n_candidates = 0;
            if (alone) hunt.level = row_results(q, h, out, r, label, xl, a);
            else part[at] = make_float4(a.m, a.s, a.u, 0.0f);
        }
        uint64_t* candidates = own_lds + maxima_words(TH, PER > 1 ? kWaveSlots : slots);  // behind the maxima
        uint32_t* orders = reinterpret_cast<uint32_t*>(candidates);  // before them
        const float bound = value_of(largest_of_lanes<DT, TH>(order_of(own), top, orders));  // a barrier inside
        meet<TH>();
        constexpr int kParts = Maxima<DT>::kParts, kRuns = kStep / kParts;
        const int each = kRuns * steps_of_slot;  // runs of a part of a slot
        const int64_t first = begin * W < q.vocab ? begin * W : q.vocab, last = end * W < q.vocab ? end * W : q.vocab;
        uint64_t* mine = keys + at * top;
        const uint32_t most = room;
        // those that reach the bound, or (above) that are over it; whether there was room for all
        const auto gather = [&](bool above) {
            for (int i = 0; i < slots; ++i) {
                const uint32_t both = tops[i * TH + lane];
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                    const float m = Maxima<DT>::get(both, part);
                    if (above ? m > bound : m >= bound) {
                        const uint32_t n = atomicAdd(&hunt.n_suspects, 1u);
                        if (n < kSuspects<TH>) hunt.suspects[n] = (uint16_t)((i * TH + lane) * kParts + part);
                    }
                }
            }
            meet<TH>();
            const uint32_t suspects = hunt.n_suspects;
            if (suspects > kSuspects<TH>) return false;
            for (int i = lane; i < (int)suspects * each; i += TH) {
                const int s = hunt.suspects[i / each], part = s % kParts, place = s / kParts / TH, who = s / kParts % TH;
                const int step = place * steps_of_slot + i % each / kRuns, of = part * kRuns + i % kRuns;
                const int64_t run = begin + who + ((int64_t)step * kStep + of) * TH, col = run * W;
                if (run >= end) continue;
                const Run<T, W> v = load_logits<DT, false>(x + col, last - col);
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    const float f = to_f32<DT>(v.e[k]);
                    if ((above ? f > bound : f >= bound) && col + k < last) {
                        const uint32_t n = atomicAdd(&hunt.n_candidates, 1u);
                        if (n < most) candidates[n] = key_of(order_of(f), (uint32_t)(col + k));
                    }
                }
            }
            meet<TH>();
            return hunt.n_candidates <= most;
        };
        bool found = a.s == a.s && gather(false);
        if (!found && a.s == a.s) {
            meet<TH>();
            if (lane == 0) hunt.n_suspects = hunt.n_candidates = 0;
            meet<TH>();
            found = gather(true);
            const uint32_t over = hunt.n_candidates;
            if (found && over < (uint32_t)top) {
                first_equal<DT, TH>(x, first, last, order_of(bound), (uint32_t)top - over, hunt.waves, candidates + over);
                meet<TH>();
                if (lane == 0) hunt.n_candidates = (uint32_t)(last - first < top ? last - first : top);
                meet<TH>();
            }
        }
        if (!found) {
            meet<TH>();
            select_keys<DT, TH>(x, first, last, top, *reinterpret_cast<Select<TH>*>(own_lds), mine);
            if (!alone) return;
            __threadfence_block();
            meet<TH>();
            for (int i = lane; i < top; i += TH) own_lds[i] = mine[i];
            meet<TH>();
            by_rank<TH>(own_lds, top, top, [&](int rank, uint64_t key) { top_result(h, out, r * top + rank, key, hunt.level); });
            return;
        }
        const int n = (int)hunt.n_candidates;
        if (alone) {
            by_rank<TH>(candidates, n, top, [&](int rank, uint64_t key) { top_result(h, out, r * top + rank, key, hunt.level); });
        } else {
            for (int i = n + lane; i < top; i += TH) mine[i] = 0;
            by_rank<TH>(candidates, n, top, [&](int rank, uint64_t key) { mine[rank] = key; });
        }
    }
}

// What the splits of rows come to: a workgroup per row with keys, else a group of lanes per row.
template <int DT, bool TOP>
__global__ __launch_bounds__(kT) void k_statistics_rows(const Rows q, const Heat h, int top, const Statistics out,
                                                        const float4* __restrict__ part, const uint64_t* __restrict__ keys,
                                                        int lanes) {
    __shared__ __align__(16) uint64_t candidates[TOP ? kMergeKeys + 2 : 1];
    __shared__ uint32_t orders[TOP ? kT : 1];
    __shared__ uint32_t count;
    __shared__ Level level_of;
    const int lane = TOP ? threadIdx.x : threadIdx.x % lanes;
    const int64_t r = TOP ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (kT / lanes) + threadIdx.x / lanes;
    if (r >= q.rows) return;
    const int64_t label = q.labels ? *gbl(q.labels + r) : 0;
    if (q.labels && label == q.ignore) return ignored_row(out, r, top, lane, TOP ? kT : lanes);
    uint64_t own[kMergeKeys / kT];
    uint64_t most = 0;
    const int n = q.splits * top;
    if constexpr (TOP) {
#pragma unroll
        for (int i = 0; i < kMergeKeys / kT; ++i) {
            const int j = i * kT + threadIdx.x;
            own[i] = j < n ? *gbl(keys + r * n + j) : 0;
            most = own[i] > most ? own[i] : most;
        }
        if (threadIdx.x == 0) count = 0;
    }
    if (!TOP || threadIdx.x < 64) {
        const float xl = label_logit<DT>(q, (const typename Elem<DT>::T*)q.x + row_offset(q, r), label);
        Sums<kEntropy> a;
        for (int i = lane; i < q.splits; i += TOP ? 64 : lanes) {
            const float4 p = part[r * q.splits + i];
            a.join(p.x, p.y, p.z, h);
        }
        wave_join(a, h, TOP ? 64 : lanes);
        if (lane == 0) {
            const Level level = row_results(q, h, out, r, label, xl, a);
            if (TOP) level_of = level;
        }
    }
    if constexpr (TOP) {
        const uint32_t bound = largest_of_lanes<DT, kT>((uint32_t)(most >> 32), top, orders);
#pragma unroll
        for (int i = 0; i < kMergeKeys / kT; ++i)
            if (own[i] != 0 && (uint32_t)(own[i] >> 32) >= bound) candidates[atomicAdd(&count, 1u)] = own[i];
        __syncthreads();
        by_rank<kT>(candidates, (int)count, top, [&](int rank, uint64_t key) { top_result(h, out, r * top + rank, key, level_of); });
    }
}

// ------------------------------------------------------------ distillation: a row's loss
struct Teacher {
    const void* ids;
    const float* logps;
    int32_t top, ids64, rest;
    float soft;      // (1 - w) tau: of d loss / d x against d D / d z
    double loss;     // (1 - w) tau^2
    double hard;     // w
};
enum { kBucket = 0, kDrop = 1, kNormalize = 2 };

__device__ __forceinline__ int64_t teacher_id(const Teacher& t, int64_t i) {
    return t.ids64 ? *gbl((const int64_t*)t.ids + i) : (int64_t)*gbl((const int32_t*)t.ids + i);
}

// What the gradient of a row needs but for its weight: e^((x - other_m) / tau) other, of the teacher's tokens
// e^((x - m) / tau) mine - soft p, and e^(x - m) plain; p = exp(log p - log_mass).
struct Slope {
    float m, other_m, mine, other, plain, log_mass, unused[2];
};

// part[row][split]: the sums of a split of a row; BUCKET: without the runs that hold a token of the teacher.  4096 x
// 128256 bf16 160 us, 6.6 TB/s: the reads, with one sum a logit beside them.
template <int DT, int U, bool BUCKET, int PER>
__global__ __launch_bounds__(kT) void k_distill(const Rows q, const Heat h, const Teacher t, float4* __restrict__ part) {
    using T = typename Elem<DT>::T;
    constexpr int TH = kT / PER, W = kW<DT>;
    __shared__ float4 waves[kT / 64];
    __shared__ uint32_t marks[BUCKET ? (PER > 1 ? PER * ((int)kShortRuns / 32 + 1) : kBits / 32) : 1];
    const int lane = threadIdx.x % TH, wave = PER > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TH) : 0;
    const int64_t at = (int64_t)blockIdx.x * PER + wave;
    const int64_t r = PER > 1 ? at : at / (uint32_t)q.splits, split = PER > 1 ? 0 : at % (uint32_t)q.splits;
    const bool counts = r < q.rows && sload(q.labels + r) != q.ignore;
    if (PER == 1 && !counts) return;
    const int64_t runs = (q.vocab + W - 1) / W, begin = split * q.split_runs;
    const int64_t end = begin + q.split_runs < runs ? begin + q.split_runs : runs;
    uint32_t* mine = marks + (PER > 1 ? wave * ((int)kShortRuns / 32 + 1) : 0);
    if constexpr (BUCKET) {
        for (int i = lane; i < (int)((end - begin + 31) / 32); i += TH) mine[i] = 0;
        __syncthreads();
        if (counts)
            for (int j = lane; j < t.top; j += TH) {
                const int64_t id = teacher_id(t, r * t.top + j);
                const int64_t run = id >= 0 && id < q.vocab ? id / W : -1;
                if (run >= begin && run < end && *gbl(t.logps + r * t.top + j) != -__builtin_inff())
                    atomicOr(&mine[(run - begin) >> 5], 1u << ((run - begin) & 31));
            }
        __syncthreads();
    }
    if (!counts) return;
    const T* x = (const T*)q.x + row_offset(q, r);
    const auto skip = [&](int64_t run) { return BUCKET && (mine[(run - begin) >> 5] >> ((run - begin) & 31) & 1); };
    const auto note = [](float, float) {};
    Sums<U> a = q.cached ? row_sums<DT, U, TH, false>(x, q.vocab, begin, end, lane, h, skip, note)
                         : row_sums<DT, U, TH, true>(x, q.vocab, begin, end, lane, h, skip, note);
    if constexpr (PER > 1) wave_join(a, h);
    else a = group_join(a, h, waves);
    if (lane == 0) part[at] = make_float4(a.m, a.s, a.u, 0.0f);
}

// What a wave finds of a row's teacher: mass and sum of p (log p - (x - ref) / tau) over its tokens (one outside of the
// vocabulary makes them NaN), ref a logit of one of them, so that large ones lose nothing, and, BUCKET, the sums over its
// tokens (each once, however many entries name it) and over what else is in their runs.
template <int U> struct Known {
    double mass, cross, log_mass, ref;
    Sums<U> tokens, others;
};

// Of one wave alone: the teacher's ids, and bits of the runs that some of them may share.
constexpr int kSeen = 16384;
template <int N> struct Named {
    int32_t ids[N];
    uint32_t seen[kSeen / 32];
};

template <int DT, int U, bool BUCKET, int N>
__device__ __forceinline__ Known<U> known_part(const Rows& q, const Heat& h, const Teacher& t, int64_t r,
                                               const typename Elem<DT>::T* x, Named<N>& own_lds) {
    using T = typename Elem<DT>::T;
    constexpr int W = kW<DT>;
    const int lane = threadIdx.x & 63;
    Known<U> o;
    o.mass = o.cross = o.log_mass = 0.0;
    Run<T, W> held_run;  // of the lane's first token
    int32_t* ids = own_lds.ids;
    bool shared = false;  // whether another token may be in the run of one of this lane's
    if constexpr (BUCKET) {
        for (int i = lane; i < kSeen / 32; i += 64) own_lds.seen[i] = 0;
        meet<64>();
    }
    float ref = 0.0f;
    for (int j0 = 0; j0 < t.top; j0 += 64) {  // every lane: the first 64 agree on ref
        const int j = j0 + lane;
        const bool there = j < t.top;
        const int64_t id = there ? teacher_id(t, r * t.top + j) : -1;
        const float lp = there ? *gbl(t.logps + r * t.top + j) : -__builtin_inff();
        const bool held = lp != -__builtin_inff(), in = id >= 0 && id < q.vocab;
        const float v = held && in ? to_f32<DT>(*gbl(x + id)) : -__builtin_inff();
        if (j0 == 0) {
            ref = v;
            for (int off = 32; off > 0; off >>= 1) ref = __builtin_fmaxf(ref, __shfl_xor(ref, off, 64));
            if (__builtin_fabsf(ref) == __builtin_inff()) ref = 0.0f;
        }
        if (there) ids[j] = held && in ? (int32_t)id : -1;
        if (!held) continue;
        const double p = in ? exp((double)lp) : __longlong_as_double(0x7ff8000000000000ll);
        o.mass += p;
        if (BUCKET && in) {
            const uint32_t bit = (uint32_t)(id / W) % kSeen;
            shared |= atomicOr(&own_lds.seen[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1;
        }
        if (BUCKET && in && j == lane) held_run = load_logits<DT, false>(x + id / W * W, q.vocab - id / W * W);
        if (p > 0.0) o.cross += p * ((double)lp - ((double)v - (double)ref) * h.inv64);
    }
    o.ref = (double)ref;
    meet<64>();
    o.mass = wave_allsum_d(o.mass);
    o.cross = wave_allsum_d(o.cross);
    if (t.rest == kNormalize) {
        // the same sum with p / mass: log p - log mass
        const bool some = !(o.mass <= 0.0);
        o.log_mass = some ? log(o.mass) : 0.0;
        o.cross = some ? o.cross / o.mass - o.log_mass : 0.0;
        o.mass = some ? o.mass / o.mass : 0.0;
    }
    if constexpr (BUCKET) {
        const int others = __ballot(shared) ? t.top : 0;
        for (int j = lane; j < t.top; j += 64) {
            const int32_t id = ids[j];
            if (id < 0) continue;
            const int32_t start = id / W * W;
            bool first = true, first_run = true;
            uint32_t named = 1u << (id - start);
#pragma unroll 4
            for (int i = 0; i < others; ++i) {
                const int32_t other = ids[i];
                const uint32_t off = (uint32_t)(other - start);  // of no token: far
                if (off < (uint32_t)W) {
                    named |= 1u << off;
                    first_run &= i >= j;
                    first &= i >= j || other != id;
                }
            }
            if (!first_run && !first) continue;
            const Run<T, W> run = j == lane ? held_run : load_logits<DT, false>(x + start, q.vocab - start);
            float own = 0.0f, top = -__builtin_inff(), v[W];
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float f = to_f32<DT>(run.e[k]);
                own = start + k == id ? f : own;
                v[k] = named >> k & 1 ? -__builtin_inff() : f;  // beyond the row's end -inf too
                top = __builtin_fmaxf(top, v[k]);
            }
            if (first) {
                o.tokens.rebase(own, h);
                o.tokens.add(own, o.tokens.base(), h);
            }
            if (!first_run) continue;
            o.others.rebase(top, h);
            const float base = o.others.base();
#pragma unroll
            for (int k = 0; k < W; ++k) o.others.add(v[k], base, h);
        }
        wave_join(o.tokens, h);
        wave_join(o.others, h);
    }
    return o;
}

// A row's loss and slope by the sums a over the logits outside of the teacher's runs (BUCKET, else over all) and the
// teacher's part, in float64: the divergence is what is left of terms that cancel.  By a whole wave: its lanes take the
// logarithms and exponentials side by side, each of which is a hundred operations.
template <int DT, int U, bool BUCKET>
__device__ __forceinline__ Slope row_slope(const Rows& q, const Heat& h, const Teacher& t, int64_t label, float label_x, Sums<U> a,
                                           const Known<U>& known, double2& each) {
    const int lane = threadIdx.x & 63;
    Sums<U> total = a;
    if constexpr (BUCKET) {
        a.join(known.others.m, known.others.s, known.others.u, h);
        total = a;
        total.join(known.tokens.m, known.tokens.s, known.tokens.u, h);
    }
    const double sum = (double)total.s, m = (double)total.m, mass = known.mass;
    const bool apart = BUCKET && a.s != 0.0f;
    const double rest = apart && mass < 1.0 ? 1.0 - mass : 0.0;
    // the teacher's tokens against the others is 1 / rho - 1; so far apart that 1 is lost: its log alone
    const double gap = ((double)known.tokens.m - (double)a.m) * h.inv64;
    double shift = 1.0, odds = 0.0;
    if (apart) {
        const double e = exp(lane == 0 ? ((double)a.m - m) * h.inv64 : fmin(gap, 600.0));
        shift = __shfl(e, 0, 64);
        odds = (double)known.tokens.s / (double)a.s * (gap > 600.0 ? 1.0 : __shfl(e, 1, 64));
    }
    const double sum1 = U == kPlain ? (double)total.u : sum;
    const double log_of = log(lane == 0 ? sum : lane == 1 ? sum1 : lane == 2 ? rest : gap > 600.0 ? odds : 1.0 + odds);
    const double log_sum = __shfl(log_of, 0, 64), log_sum1 = __shfl(log_of, 1, 64), log_rest = __shfl(log_of, 2, 64);
    const double log_odds = __shfl(log_of, 3, 64) + (gap > 600.0 ? gap : 0.0);
    const double d = known.cross + mass * ((m - known.ref) * h.inv64 + log_sum) + (rest > 0.0 ? rest * (log_rest + log_odds) : 0.0);
    // of weight 0 the teacher's part is not there, whatever it would be
    const double whole = t.soft > 0.0f ? mass + rest : 0.0, other = t.soft > 0.0f && rest > 0.0 ? rest / (double)a.s : 0.0;
    double mine = t.soft * whole / sum, others = t.soft * (whole / sum * shift - other), plain = 0.0, nll = 0.0;
    if (t.hard > 0.0) {
        const bool in = (uint64_t)label < (uint64_t)q.vocab;
        nll = in ? log_sum1 - ((double)label_x - m) : __longlong_as_double(0x7ff8000000000000ll);
        if (U == kPlain) {
            plain = t.hard / sum1;
        } else {
            mine += t.hard / sum;
            others += t.hard / sum * shift;
        }
        if (!in) mine = others = nll;
    }
    each = make_double2(d, nll);
    Slope s = {};
    s.m = total.m;
    s.other_m = apart ? a.m : total.m;
    s.mine = (float)mine;
    s.other = (float)others;
    s.plain = (float)plain;
    s.log_mass = (float)known.log_mass;
    return s;
}

// From the splits' sums of a row to its loss and slope, a wave per row: it waits for two dependent reads (8192 rows with
// 64 tokens 28 us, 48 rows 6.5 us).
template <int DT, int U, bool BUCKET>
__global__ __launch_bounds__(64) void k_distill_rows(const Rows q, const Heat h, const Teacher t, const float4* __restrict__ part,
                                                     double2* __restrict__ each, float* __restrict__ divergence,
                                                     Slope* __restrict__ slopes) {
    using T = typename Elem<DT>::T;
    __shared__ Named<kMaxTeacher> named;
    const int64_t r = blockIdx.x, label = sload(q.labels + r);
    if (label == q.ignore || (q.n_seq > 0 && seq_of(q, r) < 0)) {
        if (threadIdx.x == 0) {
            each[r] = make_double2(0.0, 0.0);
            divergence[r] = 0.0f;
        }
        return;
    }
    const T* x = (const T*)q.x + row_offset(q, r);
    const float label_x = label_logit<DT>(q, x, label);
    Sums<U> a;
    for (int i = threadIdx.x; i < q.splits; i += 64) {
        const float4 p = part[r * q.splits + i];
        a.join(p.x, p.y, p.z, h);
    }
    const Known<U> known = known_part<DT, U, BUCKET>(q, h, t, r, x, named);
    wave_join(a, h);
    double2 e;
    const Slope s = row_slope<DT, U, BUCKET>(q, h, t, label, label_x, a, known, e);
    if (threadIdx.x != 0) return;
    slopes[r] = s;
    each[r] = e;
    divergence[r] = (float)e.x;
}

struct DistillSums {
    double divergence, nll, n;
};

struct DistillTotals {
    float *loss, *divergence, *nll, *weights;
    double soft, hard;
    int32_t n_seq, parts, by_sequence;  // parts: sums to add up
};

__device__ __forceinline__ void distill_total(const DistillTotals& o, double divergence, double nll) {
    // a part of weight 0 is not there, whatever it would be
    *o.loss = (float)((o.soft != 0.0 ? o.soft * divergence : 0.0) + (o.hard != 0.0 ? o.hard * nll : 0.0));
    *o.divergence = (float)divergence;
    *o.nll = (float)nll;
}

// Sums over rows, one workgroup per sequence, or for every span of rows where there are none; one alone gives the loss
// and the weight too.  each: null where only the rows are counted.
__global__ __launch_bounds__(kSeqT) void k_distill_sums(const Rows q, const double2* __restrict__ each, DistillSums* __restrict__ sums,
                                                        int64_t span, const DistillTotals out) {
    __shared__ DistillSums waves[kSeqT / 64];
    int64_t begin = blockIdx.x * span, end = begin + span;
    if (q.n_seq > 0) {
        begin = q.cu ? (int64_t)sload(q.cu + blockIdx.x) : (int64_t)blockIdx.x * q.per_batch;
        end = q.cu ? (int64_t)sload(q.cu + blockIdx.x + 1) : begin + q.per_batch;
    }
    begin = begin < 0 ? 0 : begin;
    end = end > q.rows ? q.rows : end;
    DistillSums own = {0.0, 0.0, 0.0};
#pragma unroll 4
    for (int64_t r = begin + threadIdx.x; r < end; r += kSeqT) {
        const bool counts = *gbl(q.labels + r) != q.ignore;
        const double2 e = each ? each[r] : make_double2(0.0, 0.0);  // of every row
        own.divergence += counts ? e.x : 0.0;
        own.nll += counts ? e.y : 0.0;
        own.n += counts ? 1.0 : 0.0;
    }
    own.divergence = wave_sum_d(own.divergence);
    own.nll = wave_sum_d(own.nll);
    own.n = wave_sum_d(own.n);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = own;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < kSeqT / 64; ++w) {
        own.divergence += waves[w].divergence;
        own.nll += waves[w].nll;
        own.n += waves[w].n;
    }
    if (gridDim.x > 1) {
        sums[blockIdx.x] = own;
        return;
    }
    const double w = own.n > 0.0 ? 1.0 / own.n : 0.0;
    out.weights[0] = (float)w;
    distill_total(out, w > 0.0 ? own.divergence * w : 0.0, w > 0.0 ? own.nll * w : 0.0);
}

// Loss, means of both parts, weights per sequence, where there are several.
__global__ __launch_bounds__(kT) void k_distill_total(const DistillSums* __restrict__ sums, const DistillTotals out) {
    __shared__ double waves[kT / 64];
    double n = 0.0, seqs = 0.0;
    for (int i = threadIdx.x; i < out.parts; i += kT) {
        n += sums[i].n;
        seqs += sums[i].n > 0.0 ? 1.0 : 0.0;
    }
    n = block_sum(n, waves);
    seqs = block_sum(seqs, waves);
    double divergence = 0.0, nll = 0.0;
    for (int i = threadIdx.x; i < out.parts; i += kT) {
        const double w = sums[i].n > 0.0 ? (out.by_sequence ? 1.0 / (sums[i].n * seqs) : 1.0 / n) : 0.0;
        if (w > 0.0) {
            divergence += sums[i].divergence * w;
            nll += sums[i].nll * w;
        }
        if (out.n_seq > 0) out.weights[i] = (float)w;
    }
    divergence = block_sum(divergence, waves);
    nll = block_sum(nll, waves);
    if (threadIdx.x != 0) return;
    if (out.n_seq == 0) out.weights[0] = n > 0.0 ? (float)(1.0 / n) : 0.0f;
    distill_total(out, divergence, nll);
}

// ------------------------------------------------------------ gradients
struct Upstream {                // what the statistics' gradient takes
    const float4* stats;
    const float *logps, *entropy, *top;  // gradients; each may be null
    const int64_t* ids;
    int32_t top_n;
};
struct Downhill {                // what the distillation's takes
    const Slope* slopes;
    const float *weights, *scale_dev;
    float scale;
    Teacher t;
};

// A row's gradient: an element by its logit, and what is added at some columns.  kRuns: runs of a lane in flight, and
// all of a workgroup's; the statistics' row costs it more (4096 x 151936 bf16, 2 / 4 runs: 385 / 369 us; the
// distillation of 8192 x 128256 581 / 612).
struct StatisticsGrad {
    static constexpr int kRuns = 4;
    Upstream g;
    __device__ __forceinline__ int entries() const { return g.top ? g.top_n : 0; }
    struct Row {
        float m, log_sum, entropy, all, slope, label_extra, inv_sum;
        const float* top;
        const int64_t* ids;
        bool zero;
    };
    __device__ __forceinline__ Row row(const Rows& q, const Heat& h, int64_t r, int64_t label, int lane) const {
        Row o;
        const float4* s = g.stats + r;
        o.m = sload(&s->x);
        o.inv_sum = 1.0f / sload(&s->y);
        o.log_sum = sload(&s->z);
        o.entropy = sload(&s->w);
        o.top = g.top ? g.top + r * g.top_n : nullptr;
        o.ids = g.ids + r * g.top_n;
        const float up = g.logps ? sload(g.logps + r) * h.inv : 0.0f;
        float sum = 0.0f;
        if (g.top) {
            for (int j = lane; j < g.top_n; j += 64) sum += *gbl(o.top + j);
            sum = wave_sum(sum);
        }
        o.label_extra = up;
        o.all = -(up + sum * h.inv);
        o.slope = g.entropy ? -sload(g.entropy + r) * h.inv : 0.0f;
        if (g.logps && (uint64_t)label >= (uint64_t)q.vocab) o.all = __uint_as_float(0x7fc00000u);
        o.zero = false;
        return o;
    }
    __device__ __forceinline__ float at(const Row& o, const Heat& h, float x, bool) const {
        const float d = x - o.m, p = heat_exp(d, h) * o.inv_sum;
        const float logq = __builtin_fmaxf(d * h.inv - o.log_sum, -1e3f);  // p is 0 long before
        return p * __builtin_fmaf(o.slope, logq + o.entropy, o.all);
    }
    __device__ __forceinline__ bool entry(const Row& o, const Rows& q, const Heat& h, int j, int64_t& id, float& extra) const {
        id = *gbl(o.ids + j);
        extra = *gbl(o.top + j) * h.inv;
        return (uint64_t)id < (uint64_t)q.vocab;
    }
};

template <bool PLAIN>
struct DistillGrad {
    static constexpr int kRuns = 2;
    Downhill g;
    __device__ __forceinline__ int entries() const { return g.t.top; }
    struct Row {
        float m, other_m, mine, other, plain, log_mass, label_extra, soft;
        int64_t first;
        bool zero;
    };
    __device__ __forceinline__ float weight(const Rows& q, int64_t r) const {
        const int s = q.n_seq > 0 ? seq_of(q, r) : 0;
        return s >= 0 ? (g.scale_dev ? sload(g.scale_dev) * g.scale : g.scale) * sload(g.weights + s) : 0.0f;
    }
    __device__ __forceinline__ Row row(const Rows& q, const Heat&, int64_t r, int64_t, int) const {
        const Slope* p = g.slopes + r;
        Slope s;
        s.m = sload(&p->m);
        s.other_m = sload(&p->other_m);
        s.mine = sload(&p->mine);
        s.other = sload(&p->other);
        s.plain = sload(&p->plain);
        s.log_mass = sload(&p->log_mass);
        return row(s, weight(q, r), r);
    }
    __device__ __forceinline__ Row row(const Slope& s, float w, int64_t r) const {
        Row o;
        o.m = s.m;
        o.other_m = s.other_m;
        o.mine = s.mine * w;
        o.other = s.other * w;
        o.plain = s.plain * w;
        o.log_mass = s.log_mass;
        o.label_extra = g.t.hard > 0.0 ? -(float)g.t.hard * w : 0.0f;
        o.soft = g.t.soft * w;
        o.first = r * g.t.top;
        o.zero = w == 0.0f;
        return o;
    }
    __device__ __forceinline__ float at(const Row& o, const Heat& h, float x, bool teacher) const {
        float y = teacher ? heat_exp(x - o.m, h) * o.mine : heat_exp(x - o.other_m, h) * o.other;
        if (PLAIN) y = __builtin_fmaf(exp_(x - o.m), o.plain, y);
        return y;
    }
    __device__ __forceinline__ float extra(const Row& o, float lp) const { return g.t.soft > 0.0f ? -o.soft * exp_(lp - o.log_mass) : 0.0f; }
    __device__ __forceinline__ bool entry(const Row& o, const Rows& q, const Heat&, int j, int64_t& id, float& more) const {
        id = teacher_id(g.t, o.first + j);
        const float lp = *gbl(g.t.logps + o.first + j);
        more = extra(o, lp);
        return lp != -__builtin_inff() && (uint64_t)id < (uint64_t)q.vocab;
    }
};

// An entry at column `off` of a run v whose gradient is y: the teacher's first there changes the element's slope, each
// adds its extra.  named: the columns that have been changed.
template <int DT, class G>
__device__ __forceinline__ void take_entry(const G& g, const typename G::Row& o, const Heat& h,
                                           const Run<typename Elem<DT>::T, kW<DT>>& v, float (&y)[kW<DT>], uint32_t off, float extra,
                                           bool teacher, uint32_t& named) {
    if (teacher && !(named >> off & 1)) {
        float x = 0.0f;
#pragma unroll
        for (int k = 0; k < kW<DT>; ++k) x = (uint32_t)k == off ? to_f32<DT>(v.e[k]) : x;
        const float mine = g.at(o, h, x, true);
#pragma unroll
        for (int k = 0; k < kW<DT>; ++k) y[k] = (uint32_t)k == off ? mine : y[k];
        named |= 1u << off;
    }
#pragma unroll
    for (int k = 0; k < kW<DT>; ++k) y[k] += (uint32_t)k == off ? extra : 0.0f;
}

// The gradient of a split of a row, in runs of 16 bytes from the ends of cache lines.  Runs that hold a label or one
// of the entries are marked; the lanes that have them look through the split's list.  Bound by its bytes: of 8192 x
// 128256 bf16, 5000 rows labelled, 580 us, 5.8 TB/s of reads and writes.
template <int DT, class G, int PER>
__global__ __launch_bounds__(kT) void k_tokens_grad(const Rows q, const Heat h, const G g, void* __restrict__ grad) {
    using T = typename Elem<DT>::T;
    constexpr int TH = kT / PER, W = kW<DT>;
    constexpr int kMarks = PER > 1 ? (int)kShortRuns / 32 + 2 : kBits / 32;
    constexpr int kEntries = (PER > 1 ? kMaxTop : kMaxTeacher) + 1;
    __shared__ uint32_t marks[PER][kMarks];
    __shared__ uint32_t ids[PER][kEntries];  // highest bit: the label
    __shared__ float extras[PER][kEntries];
    __shared__ int counts[PER];
    const int lane = threadIdx.x % TH, wave = PER > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TH) : 0;
    const int64_t wg = (int64_t)blockIdx.x * PER + wave;
    const int64_t r = PER > 1 ? wg : wg / (uint32_t)q.splits, split = PER > 1 ? 0 : wg % (uint32_t)q.splits;
    const bool row = r < q.rows;
    const int64_t label = row && q.labels ? sload(q.labels + r) : 0;
    const bool learns = row && (!q.labels || label != q.ignore);
    T* out = (T*)grad + r * q.vocab;
    const Runs<W> runs(out, q.vocab, sizeof(T));
    const int64_t first = split * q.split_runs;
    int64_t end = first + q.split_runs;
    if (end > runs.count()) end = runs.count();
    int64_t c = first + lane;
    // the logits are on their way while the row's numbers and entries are found
    const T* x = (const T*)q.x + row_offset(q, r);
    Run<T, W> v[G::kRuns];
    const auto load = [&]() {
#pragma unroll
        for (int i = 0; i < G::kRuns; ++i)
            if (c + i * TH < end) v[i] = load_logits<DT>(x + runs.begin(c + i * TH), runs.left(c + i * TH));
    };
    typename G::Row o;
    o.zero = true;
    if (learns) {
        load();
        o = g.row(q, h, r, label, threadIdx.x & 63);
    }
    const bool works = learns && !o.zero;
    if (works && lane < 64) {  // in the entries' order, so that what meets at a column adds up in it
        for (int i = lane; i < (int)((end - first + 31) / 32); i += 64) marks[wave][i] = 0;
        int n = 0;
        const int all = g.entries();
        for (int j0 = 0; j0 < all + 1; j0 += 64) {
            const int j = j0 + lane;
            int64_t id = -1;
            float extra = 0.0f;
            bool in = false;
            if (j < all) in = g.entry(o, q, h, j, id, extra);
            else if (j == all && q.labels && o.label_extra != 0.0f) {
                id = label;
                extra = o.label_extra;
                in = (uint64_t)id < (uint64_t)q.vocab;
            }
            const int64_t run = in ? (id + runs.pad) / W : -1;
            in = in && run >= first && run < end;
            const uint64_t who = __ballot(in);
            if (in) {
                const int at = n + (int)__popcll(who & (((uint64_t)1 << lane) - 1));
                ids[wave][at] = (uint32_t)id | (j == all ? 0x80000000u : 0u);
                extras[wave][at] = extra;
                atomicOr(&marks[wave][(run - first) >> 5], 1u << ((run - first) & 31));
            }
            n += (int)__popcll(who);
        }
        if (lane == 0) counts[wave] = n;
    }
    if (PER > 1 || works) __syncthreads();
    if (!row) return;
    if (!works) {
        Run<T, W> zeros;
#pragma unroll
        for (int i = 0; i < W; ++i) zeros.e[i] = T(0);
        for (; c < end; c += TH) store_run<T, W>(out + runs.begin(c), runs.left(c), zeros);
        return;
    }
    const int n = counts[wave];
    for (;;) {
#pragma unroll
        for (int i = 0; i < G::kRuns; ++i) {
            const int64_t run = c + i * TH;
            if (run >= end) break;
            const int64_t at = runs.begin(run);
            float y[W];
#pragma unroll
            for (int k = 0; k < W; ++k) y[k] = g.at(o, h, to_f32<DT>(v[i].e[k]), false);
            if (marks[wave][(run - first) >> 5] >> ((run - first) & 31) & 1) {
                uint32_t named = 0;
                for (int j = 0; j < n; ++j) {
                    const uint32_t id = ids[wave][j], off = (id & 0x7fffffffu) - (uint32_t)at;
                    if (off < (uint32_t)W) take_entry<DT>(g, o, h, v[i], y, off, extras[wave][j], !(id >> 31), named);
                }
            }
#pragma unroll
            for (int k = 0; k < W; ++k) v[i].e[k] = from_f32<DT>(y[k]);
            store_run<T, W>(out + at, runs.left(run), v[i]);
        }
        c += G::kRuns * TH;
        if (c >= end) break;
        load();
    }
}

// ------------------------------------------------------------ loss and gradient of a row in one go
constexpr int kRowT = 1024;                 // threads of a workgroup that keeps a row to itself
constexpr int kKept = 4;                    // steps of a row (16 KB) that it keeps in LDS
constexpr int kRowMarks = 32768;            // runs of such a row
constexpr int kRowEntries = 2;              // of a lane: the teacher's tokens and the label

// A row by one workgroup: its sums, its loss, its gradient, where its weight is known before (the labels alone give it).
// Two workgroups a CU hold 512 rows, which the 256 MB cache still has when they are read again, last part first; the
// last steps stay in LDS between (a step in registers too spills: 8192 x 128256 bf16 all labelled, without the others'
// sum, 0 / 1 / 2 steps 844 / 895 / 976 us).  Rows of the gradient start at multiples of 16 bytes.  The first wave
// reads the teacher's tokens while the others are at the sums; in the gradient every wave holds them, a few to a lane,
// and asks by ballots which fall into its step.  8192 x 128256 bf16, 64 tokens, 5000 rows labelled: 680 us where a read
// and a write take 584, the vector units busy 65% of the time; 2406 x 32000 fp32 92 us, 5.4 TB/s.
template <int DT, bool BUCKET>
__global__ __launch_bounds__(kRowT, 8) void k_distill_alone(const Rows q, const Heat h, const DistillGrad<false> g,
                                                            double2* __restrict__ each, float* __restrict__ divergence,
                                                            Slope* __restrict__ slopes, void* __restrict__ grad) {
    using T = typename Elem<DT>::T;
    constexpr int W = kW<DT>, U = kNone;
    __shared__ float4 waves[kRowT / 64];
    __shared__ Slope slope_of;
    __shared__ uint32_t marks[BUCKET ? kRowMarks / 32 : 1];
    __shared__ Named<kRowEntries * 64> named_of;
    __shared__ Run<T, W> kept[kKept * kRowT];
    const Teacher& t = g.g.t;
    const int64_t r = blockIdx.x, label = sload(q.labels + r);
    const int lane = threadIdx.x & 63;
    T* out = (T*)grad + r * q.vocab;
    const int64_t n = q.vocab / W;
    const bool counts = label != q.ignore && (q.n_seq == 0 || seq_of(q, r) >= 0);
    Run<T, W> zeros;
#pragma unroll
    for (int i = 0; i < W; ++i) zeros.e[i] = T(0);
    if (!counts) {
        for (int64_t c = threadIdx.x; c < n; c += kRowT) store_run<T, W>(out + c * W, W, zeros);
        if (threadIdx.x == 0) {
            each[r] = make_double2(0.0, 0.0);
            divergence[r] = 0.0f;
        }
        return;
    }
    const T* x = (const T*)q.x + row_offset(q, r);
    // this lane's entries: columns (-1: none) and log-probabilities
    int32_t id[kRowEntries];
    float lp[kRowEntries];
#pragma unroll
    for (int e = 0; e < kRowEntries; ++e) {
        const int j = e * 64 + lane;
        id[e] = -1;
        lp[e] = 0.0f;
        if (j < t.top) {
            const int64_t at = teacher_id(t, r * t.top + j);
            lp[e] = *gbl(t.logps + r * t.top + j);
            if (lp[e] != -__builtin_inff() && (uint64_t)at < (uint64_t)q.vocab) id[e] = (int32_t)at;
        } else if (j == t.top && t.hard > 0.0 && (uint64_t)label < (uint64_t)q.vocab) {
            id[e] = (int32_t)label;
        }
    }
    if constexpr (BUCKET) {
        for (int i = threadIdx.x; i < kRowMarks / 32; i += kRowT) marks[i] = 0;
        __syncthreads();
        if (threadIdx.x < 64) {
#pragma unroll
            for (int e = 0; e < kRowEntries; ++e)
                if (id[e] >= 0 && e * 64 + lane < t.top) atomicOr(&marks[id[e] / W >> 5], 1u << (id[e] / W & 31));
        }
        __syncthreads();
    }
    __shared__ uint64_t known_words[sizeof(Known<U>) / 8];  // not in registers meanwhile
    Known<U>& known_of = *reinterpret_cast<Known<U>*>(known_words);
    if (threadIdx.x < 64) {
        const Known<U> known = known_part<DT, U, BUCKET>(q, h, t, r, x, named_of);
        if (threadIdx.x == 0) known_of = known;
    }
    const auto skip = [&](int64_t run) { return BUCKET && (marks[run >> 5] >> (run & 31) & 1); };
    const int64_t steps = (n + kRowT - 1) / kRowT;
    const int64_t first = steps > kKept ? steps - kKept : 0;
    const auto number = [&](int i) { return (first + i) * kRowT + threadIdx.x; };  // of kept run i
    Sums<U> a = row_sums<DT, U, kRowT, false>(x, q.vocab, 0, first * kRowT, threadIdx.x, h, skip, [](float, float) {});
    {
        LaneSums<U> end;
        const auto add = [&](const Run<T, W>& raw, int i) {
            Run<T, W> v[1] = {raw};
            if (number(i) < n && skip(number(i))) {
#pragma unroll
                for (int k = 0; k < W; ++k) v[0].e[k] = DT == F32 ? (T)-__builtin_inff() : (T)(DT == BF16 ? 0xff80 : 0xfc00);
            }
            add_runs<DT, U, 1>(end, v, largest<DT, 1>(v), h);
        };
        // what lies past the row's end reads as -inf
#pragma unroll
        for (int i = 0; i < kKept; i += 2) {
            Run<T, W> v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) v[j] = load_logits<DT>(x + number(i + j) * W, q.vocab - number(i + j) * W);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                add(v[j], i + j);
                kept[(i + j) * kRowT + threadIdx.x] = v[j];
            }
        }
        const Sums<U> b = end.sums(h);
        a.join(b.m, b.s, b.u, h);
    }
    a = group_join<U, kRowT>(a, h, waves);
    if (threadIdx.x < 64) {
        double2 e;
        const Known<U> known = known_of;
        const Slope s = row_slope<DT, U, BUCKET>(q, h, t, label, label_logit<DT>(q, x, label), a, known, e);
        if (threadIdx.x == 0) {
            slope_of = s;
            slopes[r] = s;
            each[r] = e;
            divergence[r] = (float)e.x;
        }
    }
    __syncthreads();
    const DistillGrad<false>::Row o = g.row(slope_of, g.weight(q, r), r);
    float extra_of[kRowEntries];
#pragma unroll
    for (int e = 0; e < kRowEntries; ++e) extra_of[e] = e * 64 + lane < t.top ? g.extra(o, lp[e]) : o.label_extra;
    const auto put = [&](Run<T, W> v, int64_t c) {  // c: of a wave 64 runs in a row
        if (o.zero) {
            if (c < n) store_run<T, W>(out + c * W, W, zeros);
            return;
        }
        float y[W];
#pragma unroll
        for (int k = 0; k < W; ++k) y[k] = g.at(o, h, to_f32<DT>(v.e[k]), false);
        const int32_t start = (int32_t)(c * W), step = __builtin_amdgcn_readfirstlane(start);
        uint32_t named = 0;
#pragma unroll
        for (int e = 0; e < kRowEntries; ++e) {
            uint64_t who = __ballot(id[e] >= 0 && (uint32_t)(id[e] - step) < 64u * W);
            while (who) {  // in the entries' order
                const int j = __builtin_ctzll(who);
                who &= who - 1;
                const uint32_t off = (uint32_t)(__builtin_amdgcn_readlane(id[e], j) - start);
                const float add = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(extra_of[e]), j));
                if (off < (uint32_t)W) take_entry<DT>(g, o, h, v, y, off, add, e * 64 + j < t.top, named);
            }
        }
        if (c >= n) return;
#pragma unroll
        for (int k = 0; k < W; ++k) v.e[k] = from_f32<DT>(y[k]);
        store_run<T, W>(out + c * W, W, v);
    };
#pragma unroll
    for (int i = kKept - 1; i >= 0; --i) put(kept[i * kRowT + threadIdx.x], number(i));
    // the others in pairs, one on its way while the other is written
    int64_t c = (first - 1) * kRowT + threadIdx.x;
    if (first & 1) {
        put(o.zero ? zeros : load_logits<DT>(x + c * W), c);
        c -= kRowT;
    }
    for (; c >= 0; c -= 2 * kRowT) {
        Run<T, W> v[2] = {zeros, zeros};
        if (!o.zero) {
#pragma unroll
            for (int i = 0; i < 2; ++i) v[i] = load_logits<DT>(x + (c - i * kRowT) * W);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) put(v[i], c - i * kRowT);
    }
}

// ------------------------------------------------------------ host side
int make_heat(const char* what, double temperature, Heat& h) {
    if (!(temperature >= 1e-4 && temperature <= 1e4))
        return set_error(GEFENX_EINVAL, "%s: temperature %g is not in [1e-4, 1e4]", what, temperature);
    const double c = 1.44269504088896340736 / temperature;
    h.hi = (float)c;
    if ((double)h.hi >= c) h.hi = nextafterf(h.hi, 0.0f);
    h.lo = (float)(c - (double)h.hi);
    h.inv64 = 1.0 / temperature;
    h.inv = (float)h.inv64;
    h.inv_hi = (float)(1.0 / (double)h.hi);
    h.tilt = (float)(((double)h.hi / c - 1.0) * h.inv64);
    return GEFENX_OK;
}

void set_splits(const gefenx_logits& l, Rows& q, int64_t splits) {
    const int64_t run = l.dtype == GEFENX_F32 ? 4 : 8, size = 16 / run;
    const int64_t runs = (l.vocab + kLine / size - 1 + run - 1) / run, line = kLine / 16;
    splits = std::max<int64_t>(splits, 1);
    q.split_runs = ((runs + splits - 1) / splits + line - 1) / line * line;
    q.splits = (int32_t)((runs + q.split_runs - 1) / q.split_runs);
}

// How a row is split for its sums.  A split is a round of dependent reads and joins of its own, and its results go through
// a second kernel, so rows are split only where there are fewer than two workgroups a CU and 32 passes or more, and into
// no less than 4 passes (statistics with 20 tokens, us, whole / 2 / 4 / 8 / 16 splits: 1 x 128256 bf16 20 / 18 / 15 / 13 /
// 12, 64 x 151936 23 / 21 / 17 / 16 / 18, 400 x 151936 fp32 58 / 51 / 55 / 57 / 63; 4096 x 128256 with 64 tokens 197 / 232
// / 265 in 4).  Below 32 passes the second kernel costs what the splits give (as parts of a replayed graph, whole / 2 / 4 /
// 8: 1 x 32000 bf16, 16 passes, 10.9 / 13.4 / 12.3 / 12.6, 1 x 50257, 25 passes, 12.8 / 14.9 / 13.4 / 13.0, 64 x 50257
// 14.7 / 16.3 / 14.4 / 14.3, 256 x 50257 14.8 / 19.1 / 18.4 / 22.2; 1 x 64000, 32 passes, 14.0 / 15.4 / 13.6 / 12.8).  The
// distillation has that kernel either way and takes 2-4 us longer whole there (64 x 50257 24.9 / 22.9 / 21.4 / 21.0), of
// which an eager call, 33 us of host work, shows nothing.
void split_sums(const gefenx_logits& l, Rows& q) {
    if (q.per > 1) return;
    const int64_t passes = (l.vocab * (l.dtype == GEFENX_F32 ? 4 : 2) + 16 * kT - 1) / (16 * kT);
    const int64_t wanted = (2 * kCus + q.rows - 1) / std::max<int64_t>(q.rows, 1);
    set_splits(l, q, passes < 32 ? 1 : std::min(wanted, passes / 4));
}

// How rows are split for the statistics with `top` keys a split.
int statistics_rows(const char* what, const gefenx_logits* l, int top, Rows& q) {
    if (top < 0 || top > kMaxTop) return set_error(GEFENX_EINVAL, "%s: top %d is not in [0, %d]", what, top, kMaxTop);
    const int rc = make_rows(what, l, false, q, 0, false);
    if (rc != GEFENX_OK) return rc;
    if (top > l->vocab) return set_error(GEFENX_EINVAL, "%s: top %d of %lld logits", what, top, (long long)l->vocab);
    if (top > kWaveTop) q.per = 1;
    split_sums(*l, q);
    if (top && q.splits * top > kMergeKeys) set_splits(*l, q, kMergeKeys / top);
    if ((q.rows * q.splits + q.per - 1) / q.per > kMaxThreads / kT)
        return set_error(GEFENX_EINVAL, "%s: too many rows (%lld)", what, (long long)l->rows);
    return GEFENX_OK;
}

// ... and where runs of a split are marked; most: the most passes of the gradient, 0: for the sums.
int marked_rows(const char* what, const gefenx_logits* l, bool sequences, bool labelled, int64_t most, Rows& q) {
    const int rc = make_rows(what, l, sequences, q, most, labelled);
    if (rc != GEFENX_OK) return rc;
    if (!most) split_sums(*l, q);
    if (q.split_runs > kBits) set_splits(*l, q, q.splits * ((q.split_runs + kBits - 1) / kBits) + 1);
    if (q.split_runs > kBits || (q.rows * q.splits + q.per - 1) / q.per > kMaxThreads / kT)
        return set_error(GEFENX_EINVAL, "%s: too many logits (%lld x %lld)", what, (long long)l->rows, (long long)l->vocab);
    return GEFENX_OK;
}

size_t sums_bytes(const Rows& q) { return align16(sizeof(float4) * (size_t)q.rows * (size_t)q.splits); }
size_t keys_bytes(const Rows& q, int top) { return 8 * (size_t)q.rows * (size_t)q.splits * (size_t)top; }

int enough(const char* what, const void* ws, size_t bytes, size_t needed) {
    if (!ws || bytes < needed) return set_error(GEFENX_EINVAL, "%s: workspace of %zu bytes, %zu needed", what, bytes, needed);
    return GEFENX_OK;
}

template <class G>
int run_tokens_grad(const char* what, const Rows& q, int dtype, const Heat& h, const G& g, void* grad, hipStream_t s) {
    return by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (q.per > 1) k_tokens_grad<DT, G, kT / 64><<<(uint32_t)((q.rows + q.per - 1) / q.per), kT, 0, s>>>(q, h, g, grad);
        else k_tokens_grad<DT, G, 1><<<(uint32_t)(q.rows * q.splits), kT, 0, s>>>(q, h, g, grad);
        return launched(what);
    });
}

// Workgroups that add up the rows: one per sequence; without sequences one alone as long as it is quick about it.
int sum_parts(const Rows& q) { return q.n_seq > 0 ? q.n_seq : (int)std::min<int64_t>(64, std::max<int64_t>(1, q.rows / 16384)); }

// A checked call of the distillation.
struct Distill {
    const char* what;
    Rows q;
    Heat h;
    Teacher t;
    int dtype, by_sequence;
    float4* part;
    double2* each;
    DistillSums* sums;
    float* token_divergence;
    Slope* slopes;
    DistillTotals out;
    size_t bytes;
    hipStream_t s;
};

int make_distill(const char* what, const gefenx_logits* l, const gefenx_teacher* t, int64_t most, Distill& d) {
    d.what = what;
    if (!t) return set_error(GEFENX_EINVAL, "%s: null descriptor", what);
    const int rc = marked_rows(what, l, t->by_sequence != 0 || (l && l->cu_seqlens), true, most, d.q);
    if (rc != GEFENX_OK) return rc;
    if (t->top < 1 || t->top > kMaxTeacher)
        return set_error(GEFENX_EINVAL, "%s: %d tokens of the teacher are not in [1, %d]", what, t->top, kMaxTeacher);
    if (t->rest < kBucket || t->rest > kNormalize) return set_error(GEFENX_EINVAL, "%s: rest %d", what, t->rest);
    if (!(t->hard_weight >= 0.0 && t->hard_weight <= 1.0))
        return set_error(GEFENX_EINVAL, "%s: hard_weight %g is not in [0, 1]", what, t->hard_weight);
    if (l->rows > 0 && (!t->ids || !t->logps)) return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    const int rh = make_heat(what, t->temperature, d.h);
    if (rh != GEFENX_OK) return rh;
    if (!l->cu_seqlens && !t->by_sequence) d.q.n_seq = 0;
    if (d.q.per > 1 && t->top > kMaxTop) {
        d.q.per = 1;
        set_splits(*l, d.q, 1);
        if (d.q.rows > kMaxThreads / kT) return set_error(GEFENX_EINVAL, "%s: too many rows (%lld)", what, (long long)l->rows);
    }
    d.dtype = l->dtype;
    d.by_sequence = t->by_sequence;
    d.t = Teacher{t->ids, t->logps, t->top, t->ids64, t->rest, (float)((1.0 - t->hard_weight) * t->temperature),
                  (1.0 - t->hard_weight) * t->temperature * t->temperature, t->hard_weight};
    d.bytes = sums_bytes(d.q) + sizeof(double2) * (size_t)d.q.rows + sizeof(DistillSums) * (size_t)sum_parts(d.q);
    return GEFENX_OK;
}

// The loss and the weights by the rows' results, or (each null) the weights alone.
int distill_totals(const Distill& d, const double2* each) {
    const int64_t span = (d.q.rows + d.out.parts - 1) / d.out.parts;
    k_distill_sums<<<(uint32_t)d.out.parts, kSeqT, 0, d.s>>>(d.q, each, d.sums, span, d.out);
    if (d.out.parts > 1) k_distill_total<<<1, kT, 0, d.s>>>(d.sums, d.out);
    return launched(d.what);
}

int distill_outputs(Distill& d, float* loss, float* divergence, float* nll, float* token_divergence, void* slopes, float* weights,
                    void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = d.what;
    const int rc = enough(what, workspace, workspace_bytes, d.bytes);
    if (rc != GEFENX_OK) return rc;
    if (!loss || !divergence || !nll || !weights || (d.q.rows > 0 && (!token_divergence || !slopes)))
        return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    char* ws = static_cast<char*>(workspace);
    d.part = reinterpret_cast<float4*>(ws);
    d.each = reinterpret_cast<double2*>(ws + sums_bytes(d.q));
    d.sums = reinterpret_cast<DistillSums*>(d.each + d.q.rows);
    d.s = static_cast<hipStream_t>(stream);
    d.token_divergence = token_divergence;
    d.slopes = static_cast<Slope*>(slopes);
    d.out = DistillTotals{loss, divergence, nll, weights, d.t.loss, d.t.hard, d.q.n_seq, sum_parts(d.q), d.by_sequence};
    return GEFENX_OK;
}

// go(kind of the sums, whether the teacher's other tokens count)
template <class Go>
int by_kind(const Distill& d, Go&& go) {
    using N = std::integral_constant<int, kNone>;
    using P = std::integral_constant<int, kPlain>;
    const bool plain = d.t.hard > 0.0 && d.h.inv64 != 1.0;
    if (d.t.rest == kBucket) {
        if (plain) go(P(), std::true_type());
        else go(N(), std::true_type());
    } else {
        if (plain) go(P(), std::false_type());
        else go(N(), std::false_type());
    }
    return launched(d.what);
}

int distill_forward(Distill& d) {
    const char* what = d.what;
    int rc = GEFENX_OK;
    const Rows& q = d.q;
    if (q.rows > 0) {
        rc = by_dtype(d.dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            const auto go = [&](auto u, auto bucket) {
                constexpr int U = decltype(u)::value;
                constexpr bool B = decltype(bucket)::value;
                if (q.per > 1) k_distill<DT, U, B, kT / 64><<<(uint32_t)((q.rows + q.per - 1) / q.per), kT, 0, d.s>>>(q, d.h, d.t, d.part);
                else k_distill<DT, U, B, 1><<<(uint32_t)(q.rows * q.splits), kT, 0, d.s>>>(q, d.h, d.t, d.part);
                k_distill_rows<DT, U, B><<<(uint32_t)q.rows, 64, 0, d.s>>>(q, d.h, d.t, d.part, d.each, d.token_divergence,
                                                                         d.slopes);
            };
            return by_kind(d, go);
        });
        if (rc != GEFENX_OK) return rc;
    }
    return distill_totals(d, d.each);
}

// Whether loss and gradient go row by row: rows of 96 KB or more, in rounds of two workgroups a CU that are full enough
// (32 tokens of the teacher, a fifth masked, us against two passes: bf16 256 x 128256 43 / 53, 768 x 128256 108 / 103,
// 1536 x 128256 173 / 219, 4096 x 49152 191 / 194, 8192 x 65536 436 / 464, fp32 8192 x 16384 249 / 247, 8192 x 32768
// 386 / 462).  The second exponential, where labels count at a temperature, would spill.  All rows count: how many are
// masked only the device knows.
bool rows_alone(const gefenx_logits& l, const gefenx_teacher& t, const void* grad) {
    const int64_t run = l.dtype == GEFENX_F32 ? 4 : 8, bytes = l.vocab * (16 / run);
    const bool full = l.rows >= 4 * kCus || (l.rows >= kCus && l.rows <= 2 * kCus);
    return bytes >= (96 << 10) && full && l.rows <= kMaxThreads / kRowT && l.vocab % run == 0 && l.vocab / run <= kRowMarks &&
           ((uintptr_t)grad & 15) == 0 && t.top < kRowEntries * 64 && !(t.hard_weight > 0.0 && t.temperature != 1.0);
}

int distill_alone(Distill& d, const float* scale_dev, double scale, void* grad) {
    int rc = distill_totals(d, nullptr);  // the sequences' weights come from the labels alone
    if (rc != GEFENX_OK) return rc;
    const Downhill g = {d.slopes, d.out.weights, scale_dev, (float)scale, d.t};
    rc = by_dtype(d.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const auto go = [&](auto bucket) {
            k_distill_alone<DT, decltype(bucket)::value><<<(uint32_t)d.q.rows, kRowT, 0, d.s>>>(
                d.q, d.h, DistillGrad<false>{g}, d.each, d.token_divergence, d.slopes, grad);
        };
        if (d.t.rest == kBucket) go(std::true_type());
        else go(std::false_type());
        return launched(d.what);
    });
    return rc == GEFENX_OK ? distill_totals(d, d.each) : rc;
}

int distill_grad(const char* what, const gefenx_logits* l, const gefenx_teacher* t, const void* slopes, const float* weights,
                 const float* scale_dev, double scale, void* grad, void* stream) {
    Distill d;
    const int rc = make_distill(what, l, t, DistillGrad<false>::kRuns, d);
    if (rc != GEFENX_OK || d.q.rows == 0) return rc;
    if (!slopes || !weights || !grad) return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    const Downhill g = {static_cast<const Slope*>(slopes), weights, scale_dev, (float)scale, d.t};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (d.t.hard > 0.0 && d.h.inv64 != 1.0) return run_tokens_grad(what, d.q, d.dtype, d.h, DistillGrad<true>{g}, grad, s);
    return run_tokens_grad(what, d.q, d.dtype, d.h, DistillGrad<false>{g}, grad, s);
}

}  // namespace
}  // namespace gx

using namespace gx;

extern "C" {

size_t gefenx_token_statistics_workspace_bytes(const gefenx_logits* logits, int top) {
    Rows q;
    if (statistics_rows("gefenx_token_statistics_workspace_bytes", logits, top, q) != GEFENX_OK) return 0;
    return sums_bytes(q) + keys_bytes(q, top) + 16;
}

int gefenx_token_statistics(const gefenx_logits* logits, double temperature, int top, float* logps, float* entropy,
                            int64_t* top_ids, float* top_logps, float* stats, void* workspace, size_t workspace_bytes,
                            void* stream) {
    const char* what = "gefenx_token_statistics";
    Rows q;
    Heat h;
    int rc = statistics_rows(what, logits, top, q);
    if (rc == GEFENX_OK) rc = make_heat(what, temperature, h);
    if (rc == GEFENX_OK) rc = enough(what, workspace, workspace_bytes, sums_bytes(q) + keys_bytes(q, top));
    if (rc != GEFENX_OK || q.rows == 0) return rc;
    if (!entropy || !stats || (q.labels && !logps) || (!q.labels && logps) || (top && (!top_ids || !top_logps)))
        return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float4* part = static_cast<float4*>(workspace);
    uint64_t* keys = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + sums_bytes(q));
    const Statistics out = {logps, entropy, top_logps, top_ids, reinterpret_cast<float4*>(stats)};
    return by_dtype(logits->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (top && q.per > 1) {
            const size_t lds = kT / 64 * sizeof(uint64_t) * hunt_words(64, kWaveSlots);
            k_statistics<DT, kT / 64, true><<<(uint32_t)((q.rows + q.per - 1) / q.per), kT, lds, s>>>(
                q, h, top, 1, candidates_room(64, kWaveSlots), out, part, keys);
        } else if (top) {
            constexpr int W = kW<DT>;
            const HuntPlan plan = plan_hunt(std::min(q.split_runs, (q.vocab + W - 1) / W), kT);
            k_statistics<DT, 1, true><<<(uint32_t)(q.rows * q.splits), kT, plan.bytes, s>>>(
                q, h, top, plan.steps_of_slot, plan.room, out, part, keys);
            if (q.splits > 1) k_statistics_rows<DT, true><<<(uint32_t)q.rows, kT, 0, s>>>(q, h, top, out, part, keys, 64);
        } else if (q.per > 1) {
            k_statistics<DT, kT / 64, false><<<(uint32_t)((q.rows + q.per - 1) / q.per), kT, 0, s>>>(q, h, 0, 1, 0, out, part, keys);
        } else {
            k_statistics<DT, 1, false><<<(uint32_t)(q.rows * q.splits), kT, 0, s>>>(q, h, 0, 1, 0, out, part, keys);
            int lanes = 1;
            while (lanes < q.splits && lanes < 64) lanes *= 2;
            if (q.splits > 1)
                k_statistics_rows<DT, false><<<(uint32_t)((q.rows * lanes + kT - 1) / kT), kT, 0, s>>>(q, h, 0, out, part, keys, lanes);
        }
        return launched(what);
    });
}

int gefenx_token_statistics_grad(const gefenx_logits* logits, double temperature, int top, const float* stats,
                                 const int64_t* top_ids, const float* logps_grad, const float* entropy_grad,
                                 const float* top_logps_grad, void* grad, void* stream) {
    const char* what = "gefenx_token_statistics_grad";
    Rows q;
    Heat h;
    int rc = marked_rows(what, logits, false, false, StatisticsGrad::kRuns, q);
    if (rc == GEFENX_OK) rc = make_heat(what, temperature, h);
    if (rc != GEFENX_OK) return rc;
    if (top < 0 || top > kMaxTop) return set_error(GEFENX_EINVAL, "%s: top %d is not in [0, %d]", what, top, kMaxTop);
    if (q.rows == 0) return GEFENX_OK;
    if (!stats || !grad || (top_logps_grad && !top_ids) || (logps_grad && !q.labels))
        return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    const StatisticsGrad g = {{reinterpret_cast<const float4*>(stats), logps_grad, entropy_grad, top ? top_logps_grad : nullptr,
                               top_ids, top}};
    return run_tokens_grad(what, q, logits->dtype, h, g, grad, static_cast<hipStream_t>(stream));
}

size_t gefenx_distillation_workspace_bytes(const gefenx_logits* logits, const gefenx_teacher* teacher) {
    Distill d;
    return make_distill("gefenx_distillation_workspace_bytes", logits, teacher, 0, d) == GEFENX_OK ? d.bytes + 16 : 0;
}

int gefenx_distillation_loss(const gefenx_logits* logits, const gefenx_teacher* teacher, float* loss, float* divergence,
                             float* nll, float* token_divergence, float* slopes, float* weights, void* workspace,
                             size_t workspace_bytes, void* stream) {
    Distill d;
    int rc = make_distill("gefenx_distillation_loss", logits, teacher, 0, d);
    if (rc == GEFENX_OK)
        rc = distill_outputs(d, loss, divergence, nll, token_divergence, slopes, weights, workspace, workspace_bytes, stream);
    return rc == GEFENX_OK ? distill_forward(d) : rc;
}

int gefenx_distillation_grad(const gefenx_logits* logits, const gefenx_teacher* teacher, const float* slopes,
                             const float* weights, const float* scale_dev, double scale, void* grad, void* stream) {
    return distill_grad("gefenx_distillation_grad", logits, teacher, slopes, weights, scale_dev, scale, grad, stream);
}

int gefenx_distillation_loss_grad(const gefenx_logits* logits, const gefenx_teacher* teacher, float* loss, float* divergence,
                                  float* nll, float* token_divergence, float* slopes, float* weights, const float* scale_dev,
                                  double scale, void* grad, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "gefenx_distillation_loss_grad";
    Distill d;
    int rc = make_distill(what, logits, teacher, 0, d);
    if (rc == GEFENX_OK && d.q.rows > 0 && !grad) rc = set_error(GEFENX_EINVAL, "%s: null pointer", what);
    if (rc == GEFENX_OK)
        rc = distill_outputs(d, loss, divergence, nll, token_divergence, slopes, weights, workspace, workspace_bytes, stream);
    if (rc == GEFENX_OK && rows_alone(*logits, *teacher, grad)) return distill_alone(d, scale_dev, scale, grad);
    if (rc == GEFENX_OK) rc = distill_forward(d);
    return rc == GEFENX_OK ? distill_grad(what, logits, teacher, slopes, weights, scale_dev, scale, grad, stream) : rc;
}

}  // extern "C"
