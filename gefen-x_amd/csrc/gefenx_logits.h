// gefenx_logits.h -- rows of logits: how they are split over workgroups, read and written.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gefenx.h"
#include "gefenx_device.h"
#include "gefenx_internal.h"
#include "gefenx_run.h"

namespace gx {
namespace {

constexpr int kT = 256;               // threads of a row workgroup
constexpr int64_t kWantedWgs = 2048;  // row workgroups that fill the chip: 8 on each CU
constexpr int kSeqT = 1024;           // threads of a sequence workgroup
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
// Statistics: rows are split on, to four times the workgroups that fill the chip, while each has so many
// passes: one round and a bit of long ones leaves the last CUs alone (2400 x 50257 fp32 62 -> 55 us;
// 2880 x 50257 fp16 in 8 passes each 52 against 47 whole).
constexpr int64_t kStatsPasses = 12;
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

// The sum of v over a workgroup of kT, in every lane.
__device__ __forceinline__ double block_sum(double v, double* waves) {
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < kT / 64; ++w) total += waves[w];
    return total;
}

// ------------------------------------------------------------ host side
inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GEFENX_OK : set_error(GEFENX_ELAUNCH, "%s: %s", what, hipGetErrorString(e));
}

// Row workgroups: one per row, or enough to fill the chip where the rows are few, each of a pass or
// more; `most`: the most passes of one, 0: any number; labelled: whether there have to be labels.
inline int make_rows(const char* what, const gefenx_logits* l, bool sequences, Rows& q, int64_t most = 0, bool labelled = true) {
    if (!l) return set_error(GEFENX_EINVAL, "%s: null descriptor", what);
    if (l->dtype != GEFENX_F32 && l->dtype != GEFENX_F16 && l->dtype != GEFENX_BF16)
        return set_error(GEFENX_EDTYPE, "%s: unsupported dtype %d", what, l->dtype);
    if (l->rows < 0 || l->vocab < 1 || l->rows > 0x7fffffff || l->vocab > 0x7fffffff || l->rows_per_batch < 1)
        return set_error(GEFENX_EINVAL, "%s: bad sizes (rows=%lld of %lld, vocab=%lld)", what, (long long)l->rows,
                         (long long)l->rows_per_batch, (long long)l->vocab);
    if (l->n_seq < 0 || l->n_seq > kMaxThreads / kSeqT) return set_error(GEFENX_EINVAL, "%s: bad sequences (%d)", what, l->n_seq);
    if (l->rows > 0 && (!l->logits || (labelled && !l->labels))) return set_error(GEFENX_EINVAL, "%s: null pointer", what);
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

inline size_t align16(size_t n) { return (n + 15) & ~size_t(15); }

template <class F>
int by_dtype(int dtype, F&& f) {
    switch (dtype) {
        case GEFENX_F32: return f(std::integral_constant<int, F32>());
        case GEFENX_F16: return f(std::integral_constant<int, F16>());
        default: return f(std::integral_constant<int, BF16>());
    }
}

}  // namespace
}  // namespace gx
