// What the language-model operators (embedding.cu, linear_ce.cu, clip.cu) share:
// workspaces for the time of a call, argument checks and device-side helpers.
#pragma once

#include <cstring>

#include "common.cuh"
#include "graph.cuh"

namespace mtc {

// Device error word (copy.cu) as a device address.
int device_error_word(unsigned long long **out);

// A pool block for the launches of one call on `stream`; released, in stream
// order, when the call returns (a recording keeps it for its replays).
struct Workspace {
    void *ptr = nullptr;
    cudaStream_t stream = nullptr;
    size_t used = 0;
    Workspace() = default;
    Workspace(const Workspace &) = delete;
    Workspace &operator=(const Workspace &) = delete;
    ~Workspace() { scratch_free(ptr, stream); }

    // A stream that this library does not record, but something else captures,
    // would replay into a block that the pool has handed to others by then.
    int allocate(size_t bytes, cudaStream_t s) {
        if (active_capture() == nullptr) {
            cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
            const cudaError_t e = cudaStreamIsCapturing(s, &status);
            if (e != cudaSuccess) {
                cudaGetLastError();
                return fail(MTC_ERR_RUNTIME, "the stream's capture state is unknown: %s", cudaGetErrorString(e));
            }
            if (status != cudaStreamCaptureStatusNone)
                return fail(MTC_ERR_UNSUPPORTED,
                            "this operation needs a workspace: record it with mtc_capture_begin, not on a stream "
                            "captured by other means");
        }
        stream = s;
        return scratch_alloc(bytes, s, &ptr);
    }
    // The next `bytes` of the block, on a 256-byte boundary.
    template <class T>
    T *take(size_t bytes) {
        T *p = reinterpret_cast<T *>(static_cast<char *>(ptr) + used);
        used += (bytes + 255) & ~size_t(255);
        return p;
    }
};

inline size_t padded(size_t bytes) { return (bytes + 255) & ~size_t(255); }

inline int need_float(const mtc_desc *d, const char *name) {
    MTC_TRY(validate(d, name));
    if (d->dtype != MTC_FLOAT32) return fail(MTC_ERR_INVALID_ARGUMENT, "%s must be Float32", name);
    return MTC_OK;
}

inline int need_int(const mtc_desc *d, const char *name) {
    MTC_TRY(validate(d, name));
    if (d->dtype != MTC_INT64) return fail(MTC_ERR_INVALID_ARGUMENT, "%s must be Int64", name);
    return MTC_OK;
}

// A written view gives every element its own address: no axis repeats or folds
// onto another.  Sorted by stride, each axis has to step past the ones below it.
inline int need_distinct(const mtc_desc *d, const char *name) {
    int64_t stride[MTC_MAX_RANK], extent[MTC_MAX_RANK];
    int r = 0;
    for (int i = 0; i < d->rank; ++i) {
        if (d->shape[i] == 0) return MTC_OK;
        if (d->shape[i] == 1) continue;
        const int64_t s = d->strides[i] < 0 ? -d->strides[i] : d->strides[i];
        int at = r++;
        for (; at > 0 && stride[at - 1] > s; --at) {
            stride[at] = stride[at - 1];
            extent[at] = extent[at - 1];
        }
        stride[at] = s;
        extent[at] = d->shape[i];
    }
    __int128 reach = 0;  // farthest element of the axes below
    for (int i = 0; i < r; ++i) {
        if (stride[i] <= reach)
            return fail(MTC_ERR_INVALID_ARGUMENT, "%s: elements of a written view share addresses", name);
        reach += static_cast<__int128>(stride[i]) * (extent[i] - 1);
    }
    return MTC_OK;
}

inline float *float_at(const mtc_desc *d) { return static_cast<float *>(d->data) + d->offset; }

inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

#ifdef __CUDACC__
// Launches a kernel that calls wait_for_previous() first: its CTAs may take their places while
// the kernel before it on the stream runs out, which hides most of the launch.  Only for the
// second and later kernels of a call; each of them waits for the one before, so all earlier
// ones are done as well.
template <class... P, class... A>
int launch_dependent(const char *what, void (*kernel)(P...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream,
                     A &&...args) {
    cudaLaunchAttribute attr;
    std::memset(&attr, 0, sizeof(attr));
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config;
    std::memset(&config, 0, sizeof(config));
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = &attr;
    config.numAttrs = 1;
    MTC_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...));
    return check_launch(what);
}

__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void report_index(unsigned long long *err, long long index) {
    if (atomicCAS(&err[0], 0ull, static_cast<unsigned long long>(MTC_ERR_OUT_OF_RANGE)) == 0ull)
        atomicExch(&err[1], static_cast<unsigned long long>(index));
}
#endif

}  // namespace mtc
