// What the host sides of the library's translation units share: status codes, the device of a call, launches.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

namespace dlfb200 {

// gpgpu::blas::StatusCode values used here (gpgpu/include/gblas.h:43-107)
enum : int {
    kSuccess = 0,
    kInvalidValue = -30,
    kNotImplemented = -1024,
    kInvalidMatrixA = -1022,
    kInvalidMatrixB = -1021,
    kInvalidMatrixC = -1020,
    kInvalidDimension = -1017,
    kInvalidLeadDimA = -1016,
    kInvalidLeadDimB = -1015,
    kInvalidLeadDimC = -1014,
    kInsufficientMemoryTemp = -2050,
    kInvalidBatchCount = -2049,
    kNoHalfPrecision = -2045,
    kUnexpectedError = -2039,
};

constexpr int kMaxDevices = 64;
constexpr int kSmemPerBlockOptin = 232448;  // 227 KB

#define CUDA_TRY(expr)                                   \
    do {                                                 \
        cudaError_t e__ = (expr);                        \
        if (e__ != cudaSuccess) return static_cast<int>(e__); \
    } while (0)

// The device a call works on is the one its stream belongs to (the reference binds a queue to its
// context's device, gpgpu/src/gpgpu_cu.cpp:174-204), not whatever device happens to be current on
// the calling thread. The guard makes that device current for the duration of the call and puts
// the previous one back; the legacy default stream (null) means the current device.
struct StreamDevice {
    int dev = 0;
    int prev = -1;
    int rc = kSuccess;
    explicit StreamDevice(cudaStream_t s) {
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) {
            rc = static_cast<int>(e);
            return;
        }
        if (s != nullptr && s != cudaStreamLegacy && s != cudaStreamPerThread) {
            // a stream that is being captured into a CUDA graph may not be queried (the query fails and
            // invalidates the capture): such a call works on the current device, which a capture
            // requires to be the stream's anyway
            cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
            if (cudaStreamIsCapturing(s, &cap) != cudaSuccess) {
                (void)cudaGetLastError();
                cap = cudaStreamCaptureStatusNone;
            }
            if (cap != cudaStreamCaptureStatusNone) return;
            int sd = dev;
            e = cudaStreamGetDevice(s, &sd);
            if (e != cudaSuccess) {
                rc = static_cast<int>(e);
                return;
            }
            if (sd != dev) {
                e = cudaSetDevice(sd);
                if (e != cudaSuccess) {
                    rc = static_cast<int>(e);
                    return;
                }
                prev = dev;
                dev = sd;
            }
        }
    }
    ~StreamDevice() {
        if (prev >= 0) (void)cudaSetDevice(prev);
    }
    StreamDevice(const StreamDevice&) = delete;
    StreamDevice& operator=(const StreamDevice&) = delete;
};

// A launch below is checked with cudaGetLastError(), which also returns an error that an earlier,
// unrelated runtime call of this host thread left behind (non-sticky errors stay until read).
// Such a leftover is not this call's failure: it is read away before the first launch.
inline void clear_stale_error() { (void)cudaGetLastError(); }

// launch of a programmatic dependent of the kernel before it in the stream
template <typename... Formal, typename... Actual>
cudaError_t launch_dependent(void (*kernel)(Formal...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, Actual... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Formal>(args)...);
}

// The device that is current, as the operators outside api.cu need it (set up on its first use there).
struct OperatorDevice {
    int device = 0, num_sms = 0;
    int* status = nullptr;  // the kernels' status word, read by dlf_b200_device_status
    PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
};
int operator_device(OperatorDevice* out);
unsigned tuning_bits();  // the second word of dlf_b200_set_tuning
void count_launch();

}  // namespace dlfb200
