// paged_serve.cuh — what the serving kernels of a multi-head paged cache share:
// the ragged batch, the owner of a packed token, 16-bit element conversions.
//
// Cache: K and V page arrays [n_pages][n_kv_heads][page_tokens][D] of bf16 or
// fp16 with free page / head / token strides (the last dimension contiguous).
// Batch: the new tokens of n_seq sequences packed in rows [cu_new[s],
// cu_new[s+1]); kv_len[s] tokens of sequence s are cached, the new ones among
// them, so new token j sits at position kv_len[s] - n_new[s] + j.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "heteromm_cuda.h"
#include "hmm_common.cuh"

namespace hmm {
namespace serve {

struct Batch {
    const int32_t* table;    // [n_seq][pages_per_seq]
    const int32_t* cu;       // [n_seq + 1]
    const int32_t* kv_len;   // [n_seq]
    int n_seq;
    int pages_per_seq;
    int n_tokens;            // rows of the packed batch (padding rows behind the last sequence included)
};

struct Pages {               // one page array
    unsigned char* base;
    int64_t page, head, token;   // strides in bytes
};

// One sequence of the batch.  A cu_new / kv_len entry outside its extent sets
// HMM_STATUS_BATCH_BOUNDS and makes the sequence empty (ok == false).
struct Seq {
    int begin, n_new, kv;
    bool ok;
};

__device__ __forceinline__ Seq check_seq(const Batch& b, int64_t max_kv, int begin, int end, int kv, int32_t* status) {
    Seq q;
    q.begin = begin;
    q.kv = kv;
    q.n_new = end - begin;
    q.ok = q.begin >= 0 && end >= q.begin && end <= b.n_tokens && q.kv >= 0 && q.kv <= max_kv;
    if (!q.ok) {
        atomicOr(status, HMM_STATUS_BATCH_BOUNDS);
        q.begin = q.n_new = q.kv = 0;
    }
    return q;
}

__device__ __forceinline__ Seq load_seq(const Batch& b, int64_t max_kv, int s, int32_t* status) {
    return check_seq(b, max_kv, __ldg(b.cu + s), __ldg(b.cu + s + 1), __ldg(b.kv_len + s), status);
}

// f(sequence) of every step-th sequence from s on, four sequences' loads in flight.
template <typename F>
__device__ __forceinline__ void each_seq(const Batch& b, int64_t max_kv, int s, int step, int32_t* status, F&& f) {
    for (; s < b.n_seq; s += 4 * step) {
        int begin[4], end[4], kv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = min(s + i * step, b.n_seq - 1);   // (65,535 sequences at most)
            begin[i] = __ldg(b.cu + at);
            end[i] = __ldg(b.cu + at + 1);
            kv[i] = __ldg(b.kv_len + at);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s + i * step < b.n_seq) f(check_seq(b, max_kv, begin[i], end[i], kv[i], status));
    }
}

// The last sequence s with cu[s] <= t, by one warp, 32 probes a step.  With a
// cu that is not ascending the answer is some index in [0, n_seq).
__device__ __forceinline__ int warp_find_seq(const Batch& b, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = b.n_seq;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int64_t at = (int64_t)lo + (int64_t)(lane + 1) * step;
        const bool le = at < hi && __ldg(b.cu + at) <= t;
        const int n = __popc(__ballot_sync(0xffffffffu, le));
        lo += n * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// ------------------------------------------------------------ host helpers

// Lets kernel `fn` use `bytes` of dynamic shared memory on the current device;
// `done` (static, one per kernel) remembers the devices that have been asked.
template <typename F>
hmm_status_t allow_smem(F fn, size_t bytes, std::atomic<uint64_t>* done) {
    int dev = 0;
    HMM_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (bit && (done->load(std::memory_order_relaxed) & bit)) return HMM_OK;
    HMM_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done->fetch_or(bit, std::memory_order_relaxed);
    return HMM_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Fills `b`, `k` and `v` from the ABI's descriptions, or returns the error.
hmm_status_t check_batch(const hmm_paged_cache_t* cache, const hmm_paged_batch_t* batch, Batch* b,
                         Pages* k, Pages* v);

}  // namespace serve
}  // namespace hmm
