// q4k_batch_host.h -- host-side helpers of the batch operators: a checked
// launch and a workspace that is the caller's or a stream-ordered temporary.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/q4k_batch.h"
#include "q4k_runtime.h"

namespace q4k {

template <class P>
int launch(void (*fn)(P), dim3 grid, int threads, int lds, void *stream, const P &p) {
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
