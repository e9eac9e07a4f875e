// q4k_batch.h -- what the batch operators share: a checked launch, a
// workspace that is the caller's or a stream-ordered temporary, and accesses past
// the caches.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/q4k_batch.h"
#include "q4k_runtime.h"

namespace q4k {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// F32 results of this many values and more (32 MB, the eight L2s) go past the
// caches, as what is read once for them: 4096 x 4096 values of q4k_lora_add with
// 4096 x 14336 activations 120 -> 106 us, 256 x 151936 logits 78.6 -> 74.7 us.
// Smaller ones stay for the kernel that reads them next.
constexpr int64_t kStreamFloats = 8 << 20;
// (four floats at any 4-byte aligned address)
typedef f32x4 __attribute__((aligned(4))) f32x4_any;
template <bool NT>
__device__ __forceinline__ f32x4 load4(const float *p) {
    const f32x4_any *v = reinterpret_cast<const f32x4_any *>(p);
    return NT ? __builtin_nontemporal_load(v) : *v;
}
template <bool NT>
__device__ __forceinline__ void store4(float *p, f32x4 x) {
    f32x4_any *v = reinterpret_cast<f32x4_any *>(p);
    if (NT) __builtin_nontemporal_store((f32x4_any)x, v);
    else *v = x;
}

// A launch has fewer than 2^32 threads.  (The runtime refuses more, and leaves an error that
// the next call of anyone on this thread may report as its own.)
constexpr bool launches(int64_t workgroups, int threads) { return workgroups <= (int64_t)UINT32_MAX / threads; }

template <class P>
int launch(void (*fn)(P), dim3 grid, int threads, int lds, void *stream, const P &p) {
    if (!launches(grid.x, threads)) return Q4K_EUNSUPPORTED;
    void *args[] = {const_cast<P *>(&p)};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(fn), grid, dim3((unsigned)threads), args,
                                         (size_t)lds, (hipStream_t)stream);
    return e == hipSuccess ? Q4K_OK : hip_fail(e);
}

// The caller's workspace (Q4K_EINVAL when it is too small or not 16-byte
// aligned), or a temporary that lasts until what was enqueued on the stream by
// the time of end() is done.
struct Workspace {
    void *ptr = nullptr;
    bool owned = false;

    int begin(void *workspace, size_t bytes, size_t need, void *stream) {
        if (need == 0) return Q4K_OK;
        if (workspace) {
            if (bytes < need || !aligned(workspace, 16)) return Q4K_EINVAL;
            ptr = workspace;
            return Q4K_OK;
        }
        const hipError_t e = hipMallocAsync(&ptr, need, (hipStream_t)stream);
        if (e != hipSuccess) {
            g_last_hip_error = (int32_t)e;
            return Q4K_ENOMEM;
        }
        owned = true;
        return Q4K_OK;
    }
    // the call's status: st, or that of the free
    int end(int st, void *stream) {
        if (!owned) return st;
        owned = false;
        const hipError_t e = hipFreeAsync(ptr, (hipStream_t)stream);
        return e != hipSuccess && st == Q4K_OK ? hip_fail(e) : st;
    }
};

}  // namespace q4k
