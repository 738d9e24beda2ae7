// gefenx_loss.hip -- losses over the logits of a language model, and the gradient of the logits.
//
// With l_t = x_t[y_t] - logsumexp(x_t) the log-probability of row t's label,
//   preference:  r_i = beta sum_t (l_t - ref_t),  h_j = r_j - r_{B+j},
//                loss = mean_j -(1-e) log s(h_j) - e log s(-h_j)
//   policy:      q = exp(l - old), loss = sum_t w_t (-min(q A, clip(q) A) + c (e^d - d - 1)),  d = ref - l
// and either way d loss / d x_tv = k_t ([v = y_t] - softmax(x_t)_v): a pass over the logits for the row
// statistics, a few numbers per row and sequence, and a pass that writes the gradient.  Both passes are
// bound by memory; rows without a label are not read.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gefenx.h"
#include "gefenx_device.h"
#include "gefenx_internal.h"
#include "gefenx_run.h"

namespace gx {
namespace {

constexpr int kT = 256;               // threads of a row workgroup
constexpr int64_t kWantedWgs = 2048;  // row workgroups that fill the chip: 8 on each CU
constexpr int kLine = 128;            // bytes of a cache line
// Logits up to so much are read for the statistics by ordinary loads, and the gradient finds what the 256 MB
// cache still has of them (a quarter of the rows masked, both passes: 205 MB 94.5 -> 88 us, 482 MB 200 ->
// 191; streamed loads beyond: 2.1 GB 851 against 870).
constexpr int64_t kCachedBytes = (int64_t)512 << 20;
constexpr int64_t kMaxThreads = ((int64_t)1 << 32) - 1;  // of a launch
// Rows of up to so many runs of 16 bytes go to a wave each where there are enough of them: a workgroup is
// a barrier and more than its share of lanes for them (statistics and gradient of 16384 rows, us: 1000
// bf16 logits 26.6 and 26.2 -> 12.9 and 18.6, 4096 37.6 and 58.0 -> 23.4 and 53.4; 8192, 1024 runs, 44.0
// and 102 against 43.3 and 117).
constexpr int64_t kShortRuns = 768;
// Passes of a workgroup of the gradient, and where it only writes zeros beside rows it leaves alone.  What
// is being written at any time should lie close together, and a workgroup costs its start (gradient of
// 16384 x 151936 bf16, 9216 rows labelled, 1 / 2 / 4 / 8 passes: 1490 / 1400 / 1425 / 1512 us; the whole
// policy loss on it with zeros in 1 / 2 / 4 / 8: 1650 / 1554 / 1532 / 1573).
constexpr int64_t kGradPasses = 2, kZeroPasses = 4;
// Statistics: rows are split on, to four times the workgroups that fill the chip, while each has so many
// passes: one round and a bit of long ones leaves the last CUs alone (2400 x 50257 fp32 62 -> 55 us;
// 2880 x 50257 fp16 in 8 passes each 52 against 47 whole).
constexpr int64_t kStatsPasses = 12;
constexpr int kRowT = 1024;           // threads of a workgroup that keeps a row to itself
constexpr int kKeptLds = 4, kKeptRegs = 2;  // steps of a row (16 KB) that it keeps on chip
constexpr int kSeqT = 1024;           // threads of a sequence workgroup
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eRest = (float)(1.44269504088896340736 - (double)kLog2e);

struct Rows {
    const void* x;
    const int64_t* labels;
    const int32_t* cu;
    int64_t rows, per_batch, batch_stride, row_stride;
    int64_t vocab, ignore;
    int32_t n_seq, splits;
    int32_t per, cached;   // rows of a workgroup; whether the statistics' reads are left in the cache
    int64_t split_runs;    // runs of 16 bytes of a split
};

__device__ __forceinline__ int64_t row_offset(const Rows& q, int64_t r) {
    const int64_t b = r / q.per_batch;
    return b * q.batch_stride + (r - b * q.per_batch) * q.row_stride;
}

// The sequence of row r, -1: none.
__device__ __forceinline__ int seq_of(const Rows& q, int64_t r) {
    if (!q.cu) return (int)(r / q.per_batch);
    int lo = 0, hi = q.n_seq;  // the last i with cu[i] <= r
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sload(q.cu + mid) <= r) lo = mid; else hi = mid - 1;
    }
    return lo < q.n_seq && sload(q.cu + lo) <= r ? lo : -1;
}

// Logits go 16 bytes a lane; past the end of a row -inf, which adds nothing to any sum.
template <int DT> constexpr int kW = 16 / sizeof(typename Elem<DT>::T);
template <int DT, bool STREAM = true>
__device__ __forceinline__ Run<typename Elem<DT>::T, kW<DT>> load_logits(const typename Elem<DT>::T* base, int64_t left = kW<DT>) {
    using T = typename Elem<DT>::T;
    if constexpr (DT == F32) return load_run<T, kW<DT>, STREAM>(base, left, -__builtin_inff());
    else return load_run<T, kW<DT>, STREAM>(base, left, (T)(DT == BF16 ? 0xff80 : 0xfc00));
}

// A whole run at an odd multiple of 2 bytes (every other row of an odd vocabulary, in 2-byte types):
// vectors there read at 2.4 TB/s, so the run is put together from words, each of which holds some of it.
template <int DT, bool STREAM = true>
__device__ __forceinline__ Run<typename Elem<DT>::T, kW<DT>> load_odd(const typename Elem<DT>::T* base) {
    if constexpr (DT == F32) {
        return load_logits<DT, STREAM>(base);
    } else {
        const auto a = load_run<uint32_t, 4, STREAM>(reinterpret_cast<const uint32_t*>(base - 1), 4);
        const uint32_t last = *gbl(reinterpret_cast<const uint32_t*>(base + 7));
        Run<uint32_t, 4> w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w.e[i] = __builtin_amdgcn_alignbit(i < 3 ? a.e[i + 1] : last, a.e[i], 16);
        Run<typename Elem<DT>::T, kW<DT>> r;
        __builtin_memcpy(&r, &w, sizeof(r));
        return r;
    }
}

// The runs of a row of the gradient, counted from a multiple of ALIGN bytes at or before its start, so
// that a wave's stores fill whole lines wherever the row starts.  pad: elements from there to the row.
template <int W, int ALIGN = kLine> struct Runs {
    int64_t vocab, pad;
    __device__ __forceinline__ Runs(const void* row, int64_t v, int size)
        : vocab(v), pad((int64_t)(((uintptr_t)row & (ALIGN - 1)) / size)) {}
    __device__ __forceinline__ int64_t count() const { return (vocab + pad + W - 1) / W; }
    __device__ __forceinline__ bool at_start(int64_t c) const { return c * W < pad; }  // not whole, or before the row
    __device__ __forceinline__ int64_t begin(int64_t c) const { return at_start(c) ? 0 : c * W - pad; }
    __device__ __forceinline__ int64_t left(int64_t c) const {
        const int64_t all = vocab - begin(c), within = c * W - pad + W;
        return at_start(c) && within < all ? within : all;
    }
    // runs before this one, but for those at the start, are whole
    __device__ __forceinline__ int64_t whole(int64_t end) const { return end * W <= vocab + pad ? end : end - 1; }
};

// The constant's rounding would lean every sum one way, and a sequence adds up thousands of them: its
// rest goes into the product too.
__device__ __forceinline__ float exp_(float x) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2eRest, x * kLog2e));
}

// A running maximum and the sum of exp(x - maximum).  The maximum of nothing is -inf, and -inf logits
// add 0; NaN and +inf logits make the sum NaN.
struct Soft {
    float m = -__builtin_inff(), s = 0.0f;
    __device__ __forceinline__ void rebase(float m2) {
        if (m2 > m) {
            s = s * exp_(m - m2);
            m = m2;
        }
    }
    __device__ __forceinline__ float base() const { return m == -__builtin_inff() ? 0.0f : m; }
    __device__ __forceinline__ void join(float m2, float s2) {
        const float top = m2 > m ? m2 : m;
        const float b = top == -__builtin_inff() ? 0.0f : top;
        s = s * exp_(m - b) + s2 * exp_(m2 - b);
        m = top;
    }
};

template <int DT, int N>
__device__ __forceinline__ void add_runs(Soft& a, const Run<typename Elem<DT>::T, kW<DT>> (&r)[N]) {
    float top = -__builtin_inff();
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int k = 0; k < kW<DT>; ++k) top = __builtin_fmaxf(top, to_f32<DT>(r[c].e[k]));
    a.rebase(top);
    const float b = a.base();
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int k = 0; k < kW<DT>; ++k) a.s += exp_(to_f32<DT>(r[c].e[k]) - b);
}

__device__ __forceinline__ void wave_join(Soft& a) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float m2 = __shfl_xor(a.m, off, 64), s2 = __shfl_xor(a.s, off, 64);
        a.join(m2, s2);
    }
}

// ------------------------------------------------------------ row statistics
// Runs c .. end - 1 of a row, TH lanes at a time; each lane's part.  Which logits a lane adds up, and so
// the sum, does not depend on where the row starts in memory.
template <int DT, int TH, bool STREAM>
__device__ __forceinline__ Soft row_part(const typename Elem<DT>::T* x, int64_t vocab, int64_t c, int64_t end, int lane) {
    using T = typename Elem<DT>::T;
    constexpr int W = kW<DT>;
    const int64_t whole = end * W <= vocab ? end : end - 1;
    Soft a;
    c += lane;
    const auto add = [&](auto load) {
        for (; c + 3 * TH < whole; c += 4 * TH) {
            Run<T, W> v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = load(x + (c + i * TH) * W);
            add_runs<DT, 4>(a, v);
        }
    };
    if (DT != F32 && ((uintptr_t)x & 3)) add([](const T* p) { return load_odd<DT, STREAM>(p); });
    else add([](const T* p) { return load_logits<DT, STREAM>(p); });
    for (; c < end; c += TH) {
        const Run<T, W> v[1] = {load_logits<DT, STREAM>(x + c * W, vocab - c * W)};
        add_runs<DT, 1>(a, v);
    }
    return a;
}

// The workgroup's Soft, in every lane.
template <int TH>
__device__ __forceinline__ Soft group_join(Soft a, float2* waves) {
    wave_join(a);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = make_float2(a.m, a.s);
    __syncthreads();
    a.m = waves[0].x;
    a.s = waves[0].y;
#pragma unroll
    for (int w = 1; w < TH / 64; ++w) a.join(waves[w].x, waves[w].y);
    return a;
}

// part[row][split] = {maximum, sum of exp(x - maximum)} of a split of a row.  PER rows to a workgroup:
// one, or one for each of its waves (rows without splits).  One pass with the running maximum, corrected
// once in 32 logits; a read: 9169 rows of 151936 bf16 logits 415 us, 6.7 TB/s (a read alone reaches 7.1).
template <int DT, int PER>
__global__ __launch_bounds__(kT) void k_row_stats(const Rows q, float2* __restrict__ part) {
    using T = typename Elem<DT>::T;
    constexpr int TH = kT / PER;
    __shared__ float2 waves[kT / 64];
    const int lane = threadIdx.x % TH;
    const int64_t at = (int64_t)blockIdx.x * PER + (PER > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TH) : 0);
    const int64_t r = PER > 1 ? at : at / (uint32_t)q.splits, split = PER > 1 ? 0 : at % (uint32_t)q.splits;
    if (r >= q.rows || sload(q.labels + r) == q.ignore) return;
    const int64_t runs = (q.vocab + kW<DT> - 1) / kW<DT>, begin = split * q.split_runs;
    const int64_t end = begin + q.split_runs < runs ? begin + q.split_runs : runs;
    const T* x = (const T*)q.x + row_offset(q, r);
    Soft a = q.cached ? row_part<DT, TH, false>(x, q.vocab, begin, end, lane) : row_part<DT, TH, true>(x, q.vocab, begin, end, lane);
    if constexpr (PER > 1) wave_join(a);
    else a = group_join<kT>(a, waves);
    if (lane == 0) part[at] = make_float2(a.m, a.s);
}

// ------------------------------------------------------------ tokens and sequences
struct Token {           // what the sequence kernels read and write per row
    const float* ref;    // may be null (policy without a KL term, preference without a reference)
    const float* old;
    const float* adv;    // per row or per sequence
    float* logps;
    float2* stats;       // {maximum, sum}
    float* k;            // d loss / d logp of a row but for its sequence's weight; may be null
    int32_t adv_per_row;
    float lo, hi, kl_coef;
};

struct SeqSums {         // per sequence, in float64
    double a, kl, clipped, n;
};

enum { kLogps = 0, kPreference = 1, kPolicy = 2 };

// Row r's statistics from its splits, by a group of `lanes` (a power of two, up to 64).
__device__ __forceinline__ Soft join_splits(const Rows& q, const float2* part, int64_t r, int lane, int lanes) {
    Soft a;
    for (int i = lane; i < q.splits; i += lanes) {
        const float2 p = part[r * q.splits + i];
        a.join(p.x, p.y);
    }
    for (int off = lanes >> 1; off > 0; off >>= 1) {
        const float m2 = __shfl_xor(a.m, off, 64), s2 = __shfl_xor(a.s, off, 64);
        a.join(m2, s2);
    }
    return a;
}

template <int DT>
__device__ __forceinline__ double token_logp(const Rows& q, int64_t r, int64_t label, const Soft& a) {
    using T = typename Elem<DT>::T;
    if (label < 0 || label >= q.vocab) return __longlong_as_double(0x7ff8000000000000ll);  // no such logit
    const float x = to_f32<DT>(*gbl((const T*)q.x + row_offset(q, r) + label));
    return ((double)x - (double)a.m) - log((double)a.s);
}

// A token of the policy loss: its loss, KL estimate, whether the clamped term is the minimum, and
// d loss / d logp, all but for its sequence's weight.
struct PolicyToken {
    float each, kl, k;
    bool clipped;
};
__device__ __forceinline__ PolicyToken policy_token(const Token& t, int64_t r, int64_t seq, float logp) {
    const float adv = *gbl(t.adv + (t.adv_per_row ? r : seq));
    const float ratio = expf(logp - *gbl(t.old + r));
    const float bound = __builtin_fminf(__builtin_fmaxf(ratio, t.lo), t.hi);
    const float plain = ratio * adv, clip = bound * adv;
    PolicyToken p;
    p.clipped = clip < plain;
    p.each = p.clipped ? -clip : -plain;
    p.k = p.clipped ? 0.0f : -plain;
    p.kl = 0.0f;
    if (t.ref) {
        const float d = *gbl(t.ref + r) - logp, e = expm1f(d);
        p.kl = e - d;
        p.each += t.kl_coef * p.kl;
        p.k -= t.kl_coef * e;
    }
    return p;
}

// From the rows' statistics to log-probabilities and sums: waits for a few dependent reads, 4-7 us.
// One workgroup per sequence (kLogps: per kSeqT / lanes rows), a group of lanes per row.
template <int DT, int MODE>
__global__ __launch_bounds__(kSeqT) void k_tokens(const Rows q, const Token t, const float2* __restrict__ part, int lanes,
                                                  SeqSums* __restrict__ sums) {
    __shared__ SeqSums waves[kSeqT / 64];
    const int group = threadIdx.x / lanes, lane = threadIdx.x % lanes, groups = kSeqT / lanes;
    int64_t begin, end;
    if (MODE == kLogps) {
        begin = (int64_t)blockIdx.x * groups;
        end = begin + groups;
    } else if (q.cu) {
        begin = sload(q.cu + blockIdx.x);
        end = sload(q.cu + blockIdx.x + 1);
    } else {
        begin = (int64_t)blockIdx.x * q.per_batch;
        end = begin + q.per_batch;
    }
    begin = begin < 0 ? 0 : begin;
    end = end > q.rows ? q.rows : end;
    if (MODE != kLogps && q.cu) {  // rows before the first sequence and after the last belong to none
        const int64_t first = blockIdx.x == 0 ? (begin < q.rows ? begin : q.rows) : 0;
        for (int64_t r = threadIdx.x; r < first; r += kSeqT) t.logps[r] = 0.0f;
        if (blockIdx.x + 1 == gridDim.x)
            for (int64_t r = (end > 0 ? end : 0) + threadIdx.x; r < q.rows; r += kSeqT) t.logps[r] = 0.0f;
    }
    SeqSums own = {0.0, 0.0, 0.0, 0.0};
    for (int64_t r = begin + group; r < end; r += groups) {
        const int64_t label = *gbl(q.labels + r);
        float logp = 0.0f, k = 0.0f;
        Soft a;
        if (label != q.ignore) {
            a = join_splits(q, part, r, lane, lanes);
            const double exact = token_logp<DT>(q, r, label, a);
            logp = (float)exact;
            if (MODE == kPreference && lane == 0) {
                own.a += exact - (t.ref ? (double)*gbl(t.ref + r) : 0.0);
                own.n += 1.0;
            }
            if (MODE == kPolicy && lane == 0) {
                const PolicyToken p = policy_token(t, r, blockIdx.x, logp);
                k = p.k;
                own.a += (double)p.each;
                own.kl += (double)p.kl;
                own.clipped += p.clipped ? 1.0 : 0.0;
                own.n += 1.0;
            }
        }
        if (lane == 0) {
            t.logps[r] = logp;
            t.stats[r] = make_float2(a.m, a.s);
            if (MODE == kPolicy) t.k[r] = k;
        }
    }
    if (MODE == kLogps) return;
    own.a = wave_sum_d(own.a);
    own.kl = wave_sum_d(own.kl);
    own.clipped = wave_sum_d(own.clipped);
    own.n = wave_sum_d(own.n);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = own;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kSeqT / 64; ++w) {
            own.a += waves[w].a;
            own.kl += waves[w].kl;
            own.clipped += waves[w].clipped;
            own.n += waves[w].n;
        }
        sums[blockIdx.x] = own;
    }
}

__device__ __forceinline__ double block_sum(double v, double* waves) {
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < kT / 64; ++w) total += waves[w];
    return total;
}

// The labelled rows of each sequence, and nothing else, in sums.
__global__ __launch_bounds__(kT) void k_counts(const Rows q, SeqSums* __restrict__ sums) {
    __shared__ double waves[kT / 64];
    int64_t begin = q.cu ? (int64_t)sload(q.cu + blockIdx.x) : (int64_t)blockIdx.x * q.per_batch;
    int64_t end = q.cu ? (int64_t)sload(q.cu + blockIdx.x + 1) : begin + q.per_batch;
    begin = begin < 0 ? 0 : begin;
    end = end > q.rows ? q.rows : end;
    double n = 0.0;
    for (int64_t r = begin + threadIdx.x; r < end; r += kT) n += *gbl(q.labels + r) != q.ignore ? 1.0 : 0.0;
    n = block_sum(n, waves);
    if (threadIdx.x == 0) sums[blockIdx.x] = SeqSums{0.0, 0.0, 0.0, n};
}

// Rewards of either side, and weights per sequence, the chosen ones first.
__global__ __launch_bounds__(kT) void k_preference(const SeqSums* __restrict__ sums, int n_seq, double beta, double smoothing,
                                                   int average, float* __restrict__ loss_out, float* __restrict__ chosen,
                                                   float* __restrict__ rejected, float* __restrict__ weights) {
    __shared__ double waves[kT / 64];
    const int pairs = n_seq / 2;
    double loss = 0.0;
    for (int j = threadIdx.x; j < pairs; j += kT) {
        const SeqSums c = sums[j], r = sums[pairs + j];
        const double wc = beta / (average && c.n > 0.0 ? c.n : 1.0), wr = beta / (average && r.n > 0.0 ? r.n : 1.0);
        const double h = c.a * wc - r.a * wr;
        // log s(h) = min(h, 0) - log(1 + e^-|h|); without smoothing h may be +inf
        const double tail = log1p(exp(-fabs(h)));
        loss += (1.0 - smoothing) * (tail - fmin(h, 0.0)) + (smoothing > 0.0 ? smoothing * (tail + fmax(h, 0.0)) : 0.0);
        // s(h) - (1 - e) as e - s(-h): a won pair's is all in s(-h), which 1 - s(h) would lose
        const double k = (smoothing - 1.0 / (1.0 + exp(h))) / pairs;
        chosen[j] = (float)(c.a * wc);
        rejected[j] = (float)(r.a * wr);
        weights[j] = (float)(k * wc);
        weights[pairs + j] = (float)(-k * wr);
    }
    const double total = block_sum(loss, waves);
    if (threadIdx.x == 0) *loss_out = (float)(total / pairs);
}

// Loss, mean KL, share of clipped tokens; weights per sequence.
__global__ __launch_bounds__(kT) void k_policy(const SeqSums* __restrict__ sums, int n_seq, int by_sequence,
                                               float* __restrict__ loss_out, float* __restrict__ kl_out,
                                               float* __restrict__ clipped_out, float* __restrict__ weights) {
    __shared__ double waves[kT / 64];
    double n = 0.0, seqs = 0.0, kl = 0.0, clipped = 0.0;
    for (int i = threadIdx.x; i < n_seq; i += kT) {
        n += sums[i].n;
        seqs += sums[i].n > 0.0 ? 1.0 : 0.0;
        kl += sums[i].kl;
        clipped += sums[i].clipped;
    }
    n = block_sum(n, waves);
    seqs = block_sum(seqs, waves);
    kl = block_sum(kl, waves);
    clipped = block_sum(clipped, waves);
    const double tokens = n > 0.0 ? n : 1.0;
    double loss = 0.0;
    for (int i = threadIdx.x; i < n_seq; i += kT) {
        const double w = sums[i].n > 0.0 ? (by_sequence ? 1.0 / (sums[i].n * seqs) : 1.0 / tokens) : 0.0;
        loss += sums[i].a * w;
        weights[i] = (float)w;
    }
    loss = block_sum(loss, waves);
    if (threadIdx.x == 0) {
        *loss_out = (float)loss;
        *kl_out = (float)(kl / tokens);
        *clipped_out = (float)(clipped / tokens);
    }
}

// ------------------------------------------------------------ gradient
// coef ([v = label] - exp(x - max) / sum) of a run whose first logit is number `at`, in place.
template <int DT>
__device__ __forceinline__ void grad_run(Run<typename Elem<DT>::T, kW<DT>>& v, int64_t at, int64_t label, float coef, float each,
                                         float max) {
    constexpr int W = kW<DT>;
    float g[W];
#pragma unroll
    for (int i = 0; i < W; ++i) g[i] = each * exp_(to_f32<DT>(v.e[i]) - max);
    const uint64_t here = (uint64_t)(label - at);
    if (here < W) {
#pragma unroll
        for (int i = 0; i < W; ++i) g[i] += here == (uint64_t)i ? coef : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) v.e[i] = from_f32<DT>(g[i]);
}

// grad[r][v] = c_r ([v = y_r] - exp(x - max) / sum), c_r = k[r] * weights[sequence] * scale.
// unlabelled: only the rows without a label, which get zeros.  PER: as above.  A read and a write: 8192 rows
// of 128256 bf16 logits, 4998 of them labelled, 580 us, 5.8 TB/s, a copy's rate.
template <int DT, int PER>
__global__ __launch_bounds__(kT) void k_logits_grad(const Rows q, const float2* __restrict__ stats, const float* __restrict__ k,
                                                    const float* __restrict__ weights, const float* __restrict__ scale_dev,
                                                    float scale, int unlabelled, void* __restrict__ grad) {
    using T = typename Elem<DT>::T;
    constexpr int TH = kT / PER;
    const int64_t wg = (int64_t)blockIdx.x * PER + (PER > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TH) : 0);
    const int64_t r = PER > 1 ? wg : wg / (uint32_t)q.splits, split = PER > 1 ? 0 : wg % (uint32_t)q.splits;
    if (r >= q.rows) return;
    const int64_t label = sload(q.labels + r);
    float coef = 0.0f;
    if (label != q.ignore) {
        if (unlabelled) return;
        coef = scale_dev ? sload(scale_dev) * scale : scale;
        if (k) coef *= sload(k + r);
        if (weights) {
            const int s = seq_of(q, r);
            coef = s >= 0 ? coef * sload(weights + s) : 0.0f;
            if (s >= 0 && (uint64_t)label >= (uint64_t)q.vocab) coef = __uint_as_float(0x7fc00000u);
        } else if ((uint64_t)label >= (uint64_t)q.vocab) {
            coef = __uint_as_float(0x7fc00000u);
        }
    }
    T* out = (T*)grad + r * q.vocab;
    constexpr int W = kW<DT>;
    const Runs<W> runs(out, q.vocab, sizeof(T));
    int64_t c = split * q.split_runs, end = c + q.split_runs;
    if (end > runs.count()) end = runs.count();
    const int64_t whole = runs.whole(end);
    c += threadIdx.x % TH;
    if (coef == 0.0f) {
        Run<T, W> zeros;
#pragma unroll
        for (int i = 0; i < W; ++i) zeros.e[i] = T(0);
        for (; c < end; c += TH) store_run<T, W>(out + runs.begin(c), runs.left(c), zeros);
        return;
    }
    const T* x = (const T*)q.x + row_offset(q, r);
    const float max = sload(&stats[r].x), each = -coef / sload(&stats[r].y);
    const auto one = [&](int64_t run) {
        const int64_t at = runs.begin(run), left = runs.left(run);
        Run<T, W> v = load_logits<DT>(x + at, left);
        grad_run<DT>(v, at, label, coef, each, max);
        store_run<T, W>(out + at, left, v);
    };
    if (runs.at_start(c)) {  // the first pass of a row alone: there are at most 8 such runs
        one(c);
        c += TH;
    }
    for (; c + TH < whole; c += 2 * TH) {
        Run<T, W> v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = load_logits<DT>(x + runs.begin(c + i * TH));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            grad_run<DT>(v[i], runs.begin(c + i * TH), label, coef, each, max);
            store_run<T, W>(out + runs.begin(c + i * TH), W, v[i]);
        }
    }
    for (; c < end; c += TH) one(c);
}

// Statistics and gradient of a labelled row in one go, where the coefficient needs no other row.  Two
// workgroups a CU hold 512 rows (155 MB of 151936 bf16 logits), which the 256 MB cache still has when they
// are read again, last part first.  KEEP: every row of the gradient starts at a multiple of 16 bytes, so
// both passes cut it into the same runs, and its last steps stay in LDS and registers between them (8192
// rows of 128256 bf16 logits 898 -> 847 us, of 65536 469 -> 442; two more steps in registers spill: 944).
// part[row] gets the statistics.
template <int DT, bool KEEP>
__global__ __launch_bounds__(kRowT, 2 * kRowT / 256) void k_policy_rows(const Rows q, const Token t, const float* __restrict__ weights,
                                                       const float* __restrict__ scale_dev, float scale,
                                                       float2* __restrict__ part, void* __restrict__ grad) {
    using T = typename Elem<DT>::T;
    constexpr int W = kW<DT>;
    __shared__ float2 waves[kRowT / 64];
    __shared__ float coef_of;
    __shared__ Run<T, W> kept[KEEP ? kKeptLds * kRowT : 1];
    const int64_t r = blockIdx.x, label = sload(q.labels + r);
    if (label == q.ignore) return;
    const T* x = (const T*)q.x + row_offset(q, r);
    const int64_t n = (q.vocab + W - 1) / W, steps = (n + kRowT - 1) / kRowT;
    // steps of kRowT runs: those before `first` are read twice
    constexpr int kKept = kKeptLds + kKeptRegs;
    const int64_t first = KEEP ? (steps > kKept ? steps - kKept : 0) : steps;
    const auto number = [&](int i) { return (first + i) * kRowT + threadIdx.x; };  // of kept run i
    Soft a = row_part<DT, kRowT, false>(x, q.vocab, 0, first * kRowT < n ? first * kRowT : n, threadIdx.x);
    Run<T, W> held[kKeptRegs];
    if constexpr (KEEP) {
        // what lies past the row's end reads as -inf
#pragma unroll
        for (int i = 0; i < kKeptLds; i += 2) {
            Run<T, W> v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) v[j] = load_logits<DT>(x + number(i + j) * W, q.vocab - number(i + j) * W);
            add_runs<DT, 2>(a, v);
#pragma unroll
            for (int j = 0; j < 2; ++j) kept[(i + j) * kRowT + threadIdx.x] = v[j];
        }
#pragma unroll
        for (int i = 0; i < kKeptRegs; ++i)
            held[i] = load_logits<DT>(x + number(kKeptLds + i) * W, q.vocab - number(kKeptLds + i) * W);
        add_runs<DT, kKeptRegs>(a, held);
    }
    a = group_join<kRowT>(a, waves);
    if (threadIdx.x == 0) {
        part[r] = make_float2(a.m, a.s);
        const int s = seq_of(q, r);
        float coef = 0.0f;
        if (s >= 0) {
            const float logp = (float)token_logp<DT>(q, r, label, a);
            coef = (scale_dev ? sload(scale_dev) * scale : scale) * policy_token(t, r, s, logp).k * sload(weights + s);
            if ((uint64_t)label >= (uint64_t)q.vocab) coef = __uint_as_float(0x7fc00000u);
        }
        coef_of = coef;
    }
    __syncthreads();
    const float coef = coef_of, each = -coef / a.s;
    T* out = (T*)grad + r * q.vocab;
    const Runs<W, KEEP ? 16 : kLine> runs(out, q.vocab, sizeof(T));  // KEEP: those of the first pass
    const auto put = [&](Run<T, W>& v, int64_t c) {
        const int64_t at = runs.begin(c);
        if (coef == 0.0f) {
#pragma unroll
            for (int i = 0; i < W; ++i) v.e[i] = T(0);
        } else {
            grad_run<DT>(v, at, label, coef, each, a.m);
        }
        store_run<T, W>(out + at, runs.left(c), v);
    };
    int64_t c = (runs.count() - 1) / kRowT * kRowT + threadIdx.x;
    if constexpr (KEEP) {
#pragma unroll
        for (int i = kKeptRegs - 1; i >= 0; --i) put(held[i], number(kKeptLds + i));
#pragma unroll
        for (int i = kKeptLds - 1; i >= 0; --i) {
            Run<T, W> v = kept[i * kRowT + threadIdx.x];
            put(v, number(i));
        }
        c = (first - 1) * kRowT + threadIdx.x;
    }
    for (; c >= 0; c -= kRowT) {
        if (c >= runs.count()) continue;
        Run<T, W> v;
        if (coef != 0.0f) v = load_logits<DT>(x + runs.begin(c), runs.left(c));
        put(v, c);
    }
}

// ------------------------------------------------------------ host side
int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GEFENX_OK : set_error(GEFENX_ELAUNCH, "%s: %s", what, hipGetErrorString(e));
}

// Row workgroups: one per row, or enough to fill the chip where the rows are few, each of a pass or
// more; `most`: the most passes of one, 0: any number.
int make_rows(const char* what, const gefenx_logits* l, bool sequences, Rows& q, int64_t most = 0) {
    if (!l) return set_error(GEFENX_EINVAL, "%s: null descriptor", what);
    if (l->dtype != GEFENX_F32 && l->dtype != GEFENX_F16 && l->dtype != GEFENX_BF16)
        return set_error(GEFENX_EDTYPE, "%s: unsupported dtype %d", what, l->dtype);
    if (l->rows < 0 || l->vocab < 1 || l->rows > 0x7fffffff || l->vocab > 0x7fffffff || l->rows_per_batch < 1)
        return set_error(GEFENX_EINVAL, "%s: bad sizes (rows=%lld of %lld, vocab=%lld)", what, (long long)l->rows,
                         (long long)l->rows_per_batch, (long long)l->vocab);
    if (l->n_seq < 0 || l->n_seq > kMaxThreads / kSeqT) return set_error(GEFENX_EINVAL, "%s: bad sequences (%d)", what, l->n_seq);
    if (l->rows > 0 && (!l->logits || !l->labels)) return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    if (sequences && (l->n_seq < 1 || (!l->cu_seqlens && l->rows != 0 && l->rows != l->n_seq * l->rows_per_batch)))
        return set_error(GEFENX_EINVAL, "%s: bad sequences (%d over %lld rows)", what, l->n_seq, (long long)l->rows);
    q.x = l->logits;
    q.labels = l->labels;
    q.cu = l->cu_seqlens;
    q.rows = l->rows;
    q.per_batch = l->rows_per_batch;
    q.batch_stride = l->batch_stride;
    q.row_stride = l->row_stride;
    q.vocab = l->vocab;
    q.ignore = l->ignore_index;
    q.n_seq = l->n_seq;
    const int64_t run = l->dtype == GEFENX_F32 ? 4 : 8;
    // as many as a row can have, wherever it starts
    const int64_t size = l->dtype == GEFENX_F32 ? 4 : 2, runs = (l->vocab + kLine / size - 1 + run - 1) / run;
    const int64_t passes = (runs + kT - 1) / kT;
    int64_t splits = l->rows > 0 ? (kWantedWgs + l->rows - 1) / l->rows : 1;
    if (most && splits * most < passes) splits = (passes + most - 1) / most;
    if (!most && l->rows > 0) {
        const int64_t more = (4 * kWantedWgs + l->rows - 1) / l->rows, long_enough = passes / kStatsPasses;
        splits = std::max(splits, std::min(more, long_enough));
    }
    splits = splits > passes ? passes : splits;
    if (l->rows * splits > kMaxThreads / kT) splits = kMaxThreads / kT / l->rows < 1 ? 1 : kMaxThreads / kT / l->rows;
    // workgroups meet at the ends of lines (gradient of 8 x 1024 x 128256 bf16 645 -> 580 us)
    const int64_t line = kLine / 16;
    q.split_runs = ((runs + splits - 1) / splits + line - 1) / line * line;
    q.splits = (int32_t)((runs + q.split_runs - 1) / q.split_runs);
    q.cached = l->rows * l->vocab * size <= kCachedBytes;
    q.per = runs <= kShortRuns && l->rows >= kWantedWgs ? kT / 64 : 1;
    if (q.per > 1) {
        q.splits = 1;
        q.split_runs = runs;
    }
    if ((l->rows * q.splits + q.per - 1) / q.per > kMaxThreads / kT)
        return set_error(GEFENX_EINVAL, "%s: too many rows (%lld)", what, (long long)l->rows);
    return GEFENX_OK;
}

size_t align16(size_t n) { return (n + 15) & ~size_t(15); }
size_t part_bytes(const Rows& q) { return align16(sizeof(float2) * (size_t)q.rows * (size_t)q.splits); }
size_t ws_bytes(const Rows& q) { return part_bytes(q) + sizeof(SeqSums) * (size_t)(q.n_seq > 0 ? q.n_seq : 0) + 16; }

template <class F>
int by_dtype(int dtype, F&& f) {
    switch (dtype) {
        case GEFENX_F32: return f(std::integral_constant<int, F32>());
        case GEFENX_F16: return f(std::integral_constant<int, F16>());
        default: return f(std::integral_constant<int, BF16>());
    }
}

int run_stats(const char* what, const Rows& q, int dtype, float2* part, hipStream_t s) {
    if (q.rows == 0) return GEFENX_OK;
    return by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (q.per > 1) k_row_stats<DT, kT / 64><<<(uint32_t)((q.rows + q.per - 1) / q.per), kT, 0, s>>>(q, part);
        else k_row_stats<DT, 1><<<(uint32_t)(q.rows * q.splits), kT, 0, s>>>(q, part);
        return launched(what);
    });
}

template <int MODE>
int run_tokens(const char* what, const Rows& q, int dtype, const Token& t, const float2* part, SeqSums* sums, hipStream_t s) {
    int lanes = 1;
    while (lanes < q.splits && lanes < 64) lanes *= 2;
    const int64_t wgs = MODE == kLogps ? (q.rows * lanes + kSeqT - 1) / kSeqT : q.n_seq;
    if (wgs == 0) return GEFENX_OK;
    return by_dtype(dtype, [&](auto dt) {
        k_tokens<decltype(dt)::value, MODE><<<(uint32_t)wgs, kSeqT, 0, s>>>(q, t, part, lanes, sums);
        return launched(what);
    });
}

// Whether the policy gradient goes row by row.  It reads long rows from memory once instead of twice (1.2 GB,
// few rows masked: bf16 rows of 128256 422 against 485 us, of 65536 411 against 486, fp32 rows
// of 32768 382 against 488; 1 GiB of bf16 rows of 32768 434 against 445, of 16384, which leave most of its
// 1024 lanes idle, 587 against 469).  Of fewer logits the cache still has most the second time (bf16 rows of
// 128256: 300 MB 141 against 125, 400 MB 170 against 167, 520 MB 204 against 216), and few rows are split.
// All rows count: how many are masked only the device knows.
bool rows_alone(const gefenx_logits& l) {
    const int64_t bytes = l.vocab * (l.dtype == GEFENX_F32 ? 4 : 2);
    return bytes >= (128 << 10) && l.rows >= 1024 && l.rows <= kMaxThreads / kRowT && l.rows * bytes > (int64_t)400 << 20;
}

int need(const char* what, const Rows& q, const void* ws, size_t bytes) {
    if (!ws || bytes < ws_bytes(q))
        return set_error(GEFENX_EINVAL, "%s: workspace of %zu bytes, %zu needed", what, bytes, ws_bytes(q));
    return GEFENX_OK;
}

int run_grad(const char* what, const gefenx_logits& l, const float* stats, const float* k, const float* weights,
             const float* scale_dev, double scale, int unlabelled, void* grad, hipStream_t s) {
    Rows q;
    const int rc = make_rows(what, &l, false, q, unlabelled ? kZeroPasses : kGradPasses);
    if (rc != GEFENX_OK) return rc;
    return by_dtype(l.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const float2* st = reinterpret_cast<const float2*>(stats);
        if (q.per > 1)
            k_logits_grad<DT, kT / 64><<<(uint32_t)((q.rows + q.per - 1) / q.per), kT, 0, s>>>(q, st, k, weights, scale_dev,
                                                                                             (float)scale, unlabelled, grad);
        else
            k_logits_grad<DT, 1><<<(uint32_t)(q.rows * q.splits), kT, 0, s>>>(q, st, k, weights, scale_dev, (float)scale,
                                                                              unlabelled, grad);
        return launched(what);
    });
}

// A checked call of the policy loss.
struct Policy {
    const char* what;
    Rows q;
    Token t;
    int dtype, by_sequence;
    float *loss, *kl, *clip_fraction, *weights;
    float2* part;
    SeqSums* sums;
    hipStream_t s;
};

int make_policy(const char* what, const gefenx_logits* logits, const float* old_logps, const float* advantages,
                int advantages_per_row, const float* ref_logps, double clip_low, double clip_high, double kl_coef,
                int by_sequence, float* loss, float* kl, float* clip_fraction, float* logps, float* stats, float* k,
                float* weights, void* workspace, size_t workspace_bytes, void* stream, Policy& p) {
    p.what = what;
    int rc = make_rows(what, logits, true, p.q);
    if (rc == GEFENX_OK) rc = need(what, p.q, workspace, workspace_bytes);
    if (rc != GEFENX_OK) return rc;
    if (!loss || !kl || !clip_fraction || !weights || (p.q.rows > 0 && (!logps || !stats || !k || !old_logps || !advantages)))
        return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    p.dtype = logits->dtype;
    p.by_sequence = by_sequence;
    p.loss = loss;
    p.kl = kl;
    p.clip_fraction = clip_fraction;
    p.weights = weights;
    p.part = static_cast<float2*>(workspace);
    p.sums = reinterpret_cast<SeqSums*>(static_cast<char*>(workspace) + part_bytes(p.q));
    p.s = static_cast<hipStream_t>(stream);
    p.t = Token{};
    p.t.ref = ref_logps;
    p.t.old = old_logps;
    p.t.adv = advantages;
    p.t.adv_per_row = advantages_per_row;
    p.t.logps = logps;
    p.t.stats = reinterpret_cast<float2*>(stats);
    p.t.k = k;
    p.t.lo = (float)(1.0 - clip_low);
    p.t.hi = (float)(1.0 + clip_high);
    p.t.kl_coef = (float)kl_coef;
    return GEFENX_OK;
}

// From the rows' statistics to the loss.
int policy_totals(const Policy& p) {
    const int rc = run_tokens<kPolicy>(p.what, p.q, p.dtype, p.t, p.part, p.sums, p.s);
    if (rc != GEFENX_OK) return rc;
    k_policy<<<1, kT, 0, p.s>>>(p.sums, p.q.n_seq, p.by_sequence, p.loss, p.kl, p.clip_fraction, p.weights);
    return launched(p.what);
}

}  // namespace
}  // namespace gx

using namespace gx;

extern "C" {

size_t gefenx_loss_workspace_bytes(const gefenx_logits* logits) {
    Rows q;
    return make_rows("gefenx_loss_workspace_bytes", logits, false, q) == GEFENX_OK ? ws_bytes(q) : 0;
}

int gefenx_token_logps(const gefenx_logits* logits, float* logps, float* stats, void* workspace, size_t workspace_bytes,
                       void* stream) {
    const char* what = "gefenx_token_logps";
    Rows q;
    int rc = make_rows(what, logits, false, q);
    if (rc == GEFENX_OK) rc = need(what, q, workspace, workspace_bytes);
    if (rc != GEFENX_OK) return rc;
    if (q.rows > 0 && (!logps || !stats)) return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float2* part = static_cast<float2*>(workspace);
    Token t = {};
    t.logps = logps;
    t.stats = reinterpret_cast<float2*>(stats);
    rc = run_stats(what, q, logits->dtype, part, s);
    return rc == GEFENX_OK ? run_tokens<kLogps>(what, q, logits->dtype, t, part, nullptr, s) : rc;
}

int gefenx_preference_loss(const gefenx_logits* logits, const float* ref_logps, double beta, double label_smoothing, int average,
                           float* loss, float* chosen_rewards, float* rejected_rewards, float* logps, float* stats,
                           float* weights, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "gefenx_preference_loss";
    Rows q;
    int rc = make_rows(what, logits, true, q);
    if (rc == GEFENX_OK) rc = need(what, q, workspace, workspace_bytes);
    if (rc != GEFENX_OK) return rc;
    if (q.n_seq % 2) return set_error(GEFENX_EINVAL, "%s: %d sequences are no pairs", what, q.n_seq);
    if (!loss || !chosen_rewards || !rejected_rewards || !weights || (q.rows > 0 && (!logps || !stats)))
        return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float2* part = static_cast<float2*>(workspace);
    SeqSums* sums = reinterpret_cast<SeqSums*>(static_cast<char*>(workspace) + part_bytes(q));
    Token t = {};
    t.ref = ref_logps;
    t.logps = logps;
    t.stats = reinterpret_cast<float2*>(stats);
    rc = run_stats(what, q, logits->dtype, part, s);
    if (rc == GEFENX_OK) rc = run_tokens<kPreference>(what, q, logits->dtype, t, part, sums, s);
    if (rc != GEFENX_OK) return rc;
    k_preference<<<1, kT, 0, s>>>(sums, q.n_seq, beta, label_smoothing, average, loss, chosen_rewards, rejected_rewards, weights);
    return launched(what);
}

int gefenx_policy_loss(const gefenx_logits* logits, const float* old_logps, const float* advantages, int advantages_per_row,
                       const float* ref_logps, double clip_low, double clip_high, double kl_coef, int by_sequence,
                       float* loss, float* kl, float* clip_fraction, float* logps, float* stats, float* k, float* weights,
                       void* workspace, size_t workspace_bytes, void* stream) {
    Policy p;
    int rc = make_policy("gefenx_policy_loss", logits, old_logps, advantages, advantages_per_row, ref_logps, clip_low, clip_high,
                         kl_coef, by_sequence, loss, kl, clip_fraction, logps, stats, k, weights, workspace, workspace_bytes,
                         stream, p);
    if (rc == GEFENX_OK) rc = run_stats(p.what, p.q, p.dtype, p.part, p.s);
    return rc == GEFENX_OK ? policy_totals(p) : rc;
}

int gefenx_policy_loss_grad(const gefenx_logits* logits, const float* old_logps, const float* advantages, int advantages_per_row,
                            const float* ref_logps, double clip_low, double clip_high, double kl_coef, int by_sequence,
                            float* loss, float* kl, float* clip_fraction, float* logps, float* stats, float* k, float* weights,
                            const float* scale_dev, double scale, void* grad, void* workspace, size_t workspace_bytes,
                            void* stream) {
    Policy p;
    int rc = make_policy("gefenx_policy_loss_grad", logits, old_logps, advantages, advantages_per_row, ref_logps, clip_low,
                         clip_high, kl_coef, by_sequence, loss, kl, clip_fraction, logps, stats, k, weights, workspace,
                         workspace_bytes, stream, p);
    if (rc != GEFENX_OK) return rc;
    if (p.q.rows > 0 && !grad) return set_error(GEFENX_EINVAL, "%s: null pointer", p.what);
    if (!rows_alone(*logits)) {
        rc = run_stats(p.what, p.q, p.dtype, p.part, p.s);
        if (rc == GEFENX_OK) rc = policy_totals(p);
        return rc == GEFENX_OK ? gefenx_logits_grad(logits, stats, k, weights, scale_dev, scale, grad, stream) : rc;
    }
    // the sequences' weights come from the labels alone
    k_counts<<<(uint32_t)p.q.n_seq, kT, 0, p.s>>>(p.q, p.sums);
    k_policy<<<1, kT, 0, p.s>>>(p.sums, p.q.n_seq, by_sequence, loss, kl, clip_fraction, weights);
    rc = launched(p.what);
    if (rc == GEFENX_OK) rc = run_grad(p.what, *logits, nullptr, nullptr, nullptr, nullptr, 0.0, 1, grad, p.s);
    if (rc != GEFENX_OK) return rc;
    p.q.splits = 1;
    rc = by_dtype(p.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const bool keep = ((uintptr_t)grad & 15) == 0 && p.q.vocab % kW<DT> == 0;
        const auto kernel = keep ? k_policy_rows<DT, true> : k_policy_rows<DT, false>;
        kernel<<<(uint32_t)p.q.rows, kRowT, 0, p.s>>>(p.q, p.t, weights, scale_dev, (float)scale, p.part, grad);
        return launched(p.what);
    });
    return rc == GEFENX_OK ? policy_totals(p) : rc;
}

int gefenx_logits_grad(const gefenx_logits* logits, const float* stats, const float* k, const float* weights,
                       const float* scale_dev, double scale, void* grad, void* stream) {
    const char* what = "gefenx_logits_grad";
    Rows q;
    const int rc = make_rows(what, logits, weights != nullptr, q);
    if (rc != GEFENX_OK || q.rows == 0) return rc;
    if (!stats || !grad) return set_error(GEFENX_EINVAL, "%s: null pointer", what);
    return run_grad(what, *logits, stats, k, weights, scale_dev, scale, 0, grad, static_cast<hipStream_t>(stream));
}

}  // extern "C"
