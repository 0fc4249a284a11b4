// extern "C" entries of products in 8-bit integers (declared in include/dlf_b200.h): argument checks, the choice of the
// kernel and its tile, tensor maps and launches.
#include <algorithm>
#include <climits>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include "../../include/dlf_b200.h"
#include "contraction_int8.cuh"
#include "host.cuh"
#include "quantize.cuh"

using namespace dlfb200;

namespace {

constexpr size_t kInt8MaxDepth = 131071;  // 128 * 128 * K < 2^31

int out_format(int dtype) {  // OUT_*, or -1
    return dtype == DLF_B200_HALF ? OUT_F16 : dtype == DLF_B200_BFLOAT16 ? OUT_BF16 : dtype == DLF_B200_SINGLE ? OUT_F32 : -1;
}

// ------------------------------------------------------------------------------------------------ rows to 8-bit integers

template <typename T, int WARPS, int PIECES>
int quantize_launch(const QuantizeParams& p, cudaStream_t stream) {
    constexpr int kRows = kQuantizeThreads / 32 / WARPS;
    const unsigned grid = static_cast<unsigned>((p.rows + kRows - 1) / kRows);
    CUDA_TRY(launch_dependent(quantize_rows_kernel<T, WARPS, PIECES>, grid, kQuantizeThreads, 0, stream, p));
    count_launch();
    CUDA_TRY(cudaGetLastError());
    return kSuccess;
}

template <typename T>
int quantize_any(const QuantizeParams& p, int num_sms, cudaStream_t stream) {
    const long long pieces = (p.cols + 7) / 8;
    // a warp for a row where that still gives every SM some, else a block for a row
    if (pieces <= 32 * 8 && p.rows >= 16ll * num_sms) {
        if (pieces <= 32) return quantize_launch<T, 1, 1>(p, stream);
        if (pieces <= 64) return quantize_launch<T, 1, 2>(p, stream);
        if (pieces <= 128) return quantize_launch<T, 1, 4>(p, stream);
        return quantize_launch<T, 1, 8>(p, stream);
    }
    if (pieces <= 256) return quantize_launch<T, 8, 1>(p, stream);
    if (pieces <= 512) return quantize_launch<T, 8, 2>(p, stream);
    if (pieces <= 1024) return quantize_launch<T, 8, 4>(p, stream);
    if (pieces <= 2048) return quantize_launch<T, 8, 8>(p, stream);
    return quantize_launch<T, 8, 0>(p, stream);
}

// ------------------------------------------------------------------------------------------------ products

struct Int8Problem {
    int out;
    long long M, N, K;
    const signed char* a;
    long long a_ld;
    const float* sa;
    const signed char* b;
    long long b_ld;
    const float* sb;
    const char* bias;
    int relu;
    char* d;
    long long ldd;
};

bool lines_aligned(const signed char* base, long long ld, long long lines) {
    return (reinterpret_cast<uintptr_t>(base) & 15u) == 0 && (lines == 1 || ld % 16 == 0) && ld < (1ll << 40);
}

int encode_int8(const OperatorDevice& dev, CUtensorMap* map, const signed char* base, long long ld, long long lines, long long K, int box_lines) {
    const cuuint64_t pitch = ld % 16 == 0 && ld > 0 ? static_cast<cuuint64_t>(ld) : static_cast<cuuint64_t>((K + 15) / 16 * 16);  // (one line: any)
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(lines), 1};
    cuuint64_t strides[2] = {pitch, pitch};
    cuuint32_t box[3] = {128, static_cast<cuuint32_t>(box_lines), 1}, estr[3] = {1, 1, 1};
    const CUresult r = dev.encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<signed char*>(base), dims, strides, box, estr,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? kSuccess : kUnexpectedError;
}

struct Int8Device {
    bool ready = false;
    int max_pairs = 0;  // co-resident CTA pairs of int8_pair_kernel
};
Int8Device g_int8[kMaxDevices];
std::mutex g_int8_mu;

template <int OUT, bool CHANNELS>
int int8_tile_limits() {
    CUDA_TRY(cudaFuncSetAttribute(int8_tile_kernel<OUT, CHANNELS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerBlockOptin - 1024));
    return kSuccess;
}

template <int OUT>
int int8_pair_limits(int num_sms, int* pairs) {
    CUDA_TRY(cudaFuncSetAttribute(int8_pair_kernel<OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kInt8PairSmem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * num_sms), 1, 1);
    cfg.blockDim = dim3(kInt8PairThreads, 1, 1);
    cfg.dynamicSmemBytes = kInt8PairSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CUDA_TRY(cudaOccupancyMaxActiveClusters(pairs, int8_pair_kernel<OUT>, &cfg));
    return *pairs > 0 ? kSuccess : kUnexpectedError;
}

int int8_device(const OperatorDevice& dev, int* max_pairs) {
    std::lock_guard<std::mutex> lock(g_int8_mu);
    Int8Device& st = g_int8[dev.device];
    if (st.ready) {
        *max_pairs = st.max_pairs;
        return kSuccess;
    }
    for (int rc : {int8_pair_limits<OUT_F32>(dev.num_sms, &st.max_pairs), int8_pair_limits<OUT_F16>(dev.num_sms, &st.max_pairs),
                   int8_pair_limits<OUT_BF16>(dev.num_sms, &st.max_pairs)})
        if (rc != kSuccess) return rc;
    *max_pairs = st.max_pairs;
    for (int rc : {int8_tile_limits<OUT_F32, false>(), int8_tile_limits<OUT_F16, false>(), int8_tile_limits<OUT_BF16, false>(),
                   int8_tile_limits<OUT_F32, true>(), int8_tile_limits<OUT_F16, true>(), int8_tile_limits<OUT_BF16, true>()})
        if (rc != kSuccess) return rc;
    st.ready = true;
    return kSuccess;
}

template <bool CHANNELS>
int int8_tile_launch(const OperatorDevice& dev, const Int8Problem& q, cudaStream_t stream) {
    Int8Params p{};
    const long long lanes = CHANNELS ? q.N : q.M, cols = CHANNELS ? q.M : q.N;
    p.BN = cols <= 16 ? 16 : cols <= 32 ? 32 : cols <= 64 ? 64 : 128;
    const long long tiles_l = (lanes + kBM - 1) / kBM, tiles_c = (cols + p.BN - 1) / p.BN, tiles = tiles_l * tiles_c;
    const long long num_kb = (q.K + 127) / 128;
    p.S = 1;
    while (2 * p.S <= kSplitMaxCtas && tiles * 2 * p.S <= dev.num_sms && num_kb >= 4 * p.S) p.S *= 2;
    if (tiles * p.S > INT_MAX) return kInvalidDimension;
    const int stage = (kBM + p.BN) * 128;
    p.stages = static_cast<int>(std::min<long long>({static_cast<long long>(kInt8MaxStages), (num_kb + p.S - 1) / p.S, (kSmemPerBlockOptin - 2048) / stage}));
    p.M = static_cast<int>(q.M);
    p.N = static_cast<int>(q.N);
    p.K = static_cast<int>(q.K);
    p.tiles_l = static_cast<int>(tiles_l);
    p.tiles_c = static_cast<int>(tiles_c);
    p.sa = q.sa;
    p.sb = q.sb;
    p.bias = q.bias;
    p.relu = q.relu;
    p.d = q.d;
    p.ldd = q.ldd;
    const int es = q.out == OUT_F32 ? 4 : 2;
    p.vec = (reinterpret_cast<uintptr_t>(q.d) % (4 * es) == 0 && q.ldd % 4 == 0) ? 1 : 0;
    p.status = dev.status;
    const bool inject = (tuning_bits() & 0x10000000u) != 0 && tiles == 1;
    p.wait_limit = inject ? (1ll << 21) : (1ll << 32);
    p.withhold = inject ? 1 : 0;
    CUtensorMap tm_a, tm_b;
    int rc = encode_int8(dev, &tm_a, q.a, q.a_ld, q.M, q.K, CHANNELS ? p.BN : kBM);
    if (rc != kSuccess) return rc;
    rc = encode_int8(dev, &tm_b, q.b, q.b_ld, q.N, q.K, CHANNELS ? kBM : p.BN);
    if (rc != kSuccess) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * p.S), 1, 1);
    cfg.blockDim = dim3(kInt8Threads, 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(int8_tile_smem(p.BN, p.stages));
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(p.S);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.S > 1 ? 2 : 1;
    const CUtensorMap& tl = CHANNELS ? tm_b : tm_a;
    const CUtensorMap& tc = CHANNELS ? tm_a : tm_b;
    if (q.out == OUT_F32) CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_tile_kernel<OUT_F32, CHANNELS>, p, tl, tc));
    else if (q.out == OUT_F16) CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_tile_kernel<OUT_F16, CHANNELS>, p, tl, tc));
    else CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_tile_kernel<OUT_BF16, CHANNELS>, p, tl, tc));
    count_launch();
    CUDA_TRY(cudaGetLastError());
    return kSuccess;
}

int int8_pair_launch(const OperatorDevice& dev, int max_pairs, const Int8Problem& q, cudaStream_t stream) {
    Int8Params p{};
    p.M = static_cast<int>(q.M);
    p.N = static_cast<int>(q.N);
    p.K = static_cast<int>(q.K);
    const long long tiles_l = (q.M + 2 * kBM - 1) / (2 * kBM), tiles_c = (q.N + kInt8PairBN - 1) / kInt8PairBN, tiles = tiles_l * tiles_c;
    if (tiles > INT_MAX / 16) return kInvalidDimension;
    p.tiles_l = static_cast<int>(tiles_l);
    p.tiles_c = static_cast<int>(tiles_c);
    p.sa = q.sa;
    p.sb = q.sb;
    p.bias = q.bias;
    p.relu = q.relu;
    p.d = q.d;
    p.ldd = q.ldd;
    const int es = q.out == OUT_F32 ? 4 : 2;
    // TMA stores are clipped at the next 16-byte boundary past a line's end, so the lines must end on one
    p.vec = (reinterpret_cast<uintptr_t>(q.d) % 16 == 0 && q.ldd * es % 16 == 0 && q.N * es % 16 == 0 && q.ldd * es < (1ll << 40)) ? 1 : 0;
    p.status = dev.status;
    p.wait_limit = 1ll << 32;
    CUtensorMap tm_a, tm_b, tm_d;
    int rc = encode_int8(dev, &tm_a, q.a, q.a_ld, q.M, q.K, kBM);
    if (rc != kSuccess) return rc;
    rc = encode_int8(dev, &tm_b, q.b, q.b_ld, q.N, q.K, kBM);
    if (rc != kSuccess) return rc;
    tm_d = tm_a;
    if (p.vec) {
        cuuint64_t dims[3] = {static_cast<cuuint64_t>(q.N), static_cast<cuuint64_t>(q.M), 1};
        cuuint64_t strides[2] = {static_cast<cuuint64_t>(q.ldd * es), static_cast<cuuint64_t>(q.ldd * es)};
        cuuint32_t box[3] = {static_cast<cuuint32_t>(128 / es), 32, 1}, estr[3] = {1, 1, 1};
        if (dev.encode(&tm_d, es == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, q.d, dims, strides, box, estr,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return kUnexpectedError;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<long long>(tiles, max_pairs)), 1, 1);
    cfg.blockDim = dim3(kInt8PairThreads, 1, 1);
    cfg.dynamicSmemBytes = kInt8PairSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (q.out == OUT_F32) CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_pair_kernel<OUT_F32>, p, tm_a, tm_b, tm_d));
    else if (q.out == OUT_F16) CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_pair_kernel<OUT_F16>, p, tm_a, tm_b, tm_d));
    else CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_pair_kernel<OUT_BF16>, p, tm_a, tm_b, tm_d));
    count_launch();
    CUDA_TRY(cudaGetLastError());
    return kSuccess;
}

// Operands whose lines start off 16-byte boundaries are copied into the caller's scratch first.
size_t padded_depth(size_t k) { return (k + 15) / 16 * 16; }

size_t int8_copy_bytes(size_t m, size_t n, size_t k, const signed char* a, size_t a_ld, const signed char* b, size_t b_ld) {
    size_t bytes = 0;
    if (!lines_aligned(a, static_cast<long long>(a_ld), static_cast<long long>(m))) bytes += m * padded_depth(k);
    if (!lines_aligned(b, static_cast<long long>(b_ld), static_cast<long long>(n))) bytes += n * padded_depth(k);
    return bytes == 0 ? 0 : bytes + 256;
}

int int8_copy(const OperatorDevice& dev, Int8Problem& q, char* ws, cudaStream_t stream) {
    Int8Lines p{};
    int n = 0;
    long long most = 0;
    signed char* to = reinterpret_cast<signed char*>((reinterpret_cast<uintptr_t>(ws) + 255) / 256 * 256);
    p.length = static_cast<int>(q.K);
    p.dst_pitch = static_cast<int>(padded_depth(static_cast<size_t>(q.K)));
    auto add = [&](const signed char*& base, long long& ld, long long lines) {
        if (lines_aligned(base, ld, lines)) return;
        p.src[n] = base;
        p.src_pitch[n] = ld;
        p.dst[n] = to;
        p.lines[n] = lines;
        most = std::max(most, lines * p.dst_pitch / 16);
        base = to;
        ld = p.dst_pitch;
        to += lines * p.dst_pitch;
        ++n;
    };
    add(q.a, q.a_ld, q.M);
    add(q.b, q.b_ld, q.N);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<long long>((most + 255) / 256, 8ll * dev.num_sms)), static_cast<unsigned>(n), 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_lines_kernel, p));
    count_launch();
    CUDA_TRY(cudaGetLastError());
    return kSuccess;
}

}  // namespace

extern "C" {

int dlf_b200_quantize_rows(int dtype, size_t rows, size_t cols, const void* x, size_t x_ld, signed char* q, size_t q_ld, float* scales,
                           void* stream) {
    if (out_format(dtype) < 0) return kNotImplemented;
    if (rows == 0 || cols == 0 || rows > INT_MAX || cols > INT_MAX) return kInvalidDimension;
    if (x_ld < cols) return kInvalidLeadDimA;
    if (q_ld < cols) return kInvalidLeadDimC;
    if (x == nullptr) return kInvalidMatrixA;
    if (q == nullptr || scales == nullptr) return kInvalidMatrixC;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    StreamDevice guard(s);
    if (guard.rc != kSuccess) return guard.rc;
    OperatorDevice dev;
    const int rc = operator_device(&dev);
    if (rc != kSuccess) return rc;
    clear_stale_error();
    QuantizeParams p{static_cast<const char*>(x), static_cast<long long>(x_ld), q, static_cast<long long>(q_ld), scales,
                     static_cast<long long>(rows), static_cast<long long>(cols)};
    if (dtype == DLF_B200_HALF) return quantize_any<__half>(p, dev.num_sms, s);
    if (dtype == DLF_B200_BFLOAT16) return quantize_any<__nv_bfloat16>(p, dev.num_sms, s);
    return quantize_any<float>(p, dev.num_sms, s);
}

size_t dlf_b200_gemm_int8_workspace_bytes(size_t m, size_t n, size_t k, const signed char* a, size_t a_ld, const signed char* b, size_t b_ld) {
    return int8_copy_bytes(m, n, k, a, a_ld, b, b_ld);
}

int dlf_b200_gemm_int8(int dtype, size_t m, size_t n, size_t k, const signed char* a, size_t a_ld, const float* a_scales,
                       const signed char* b, size_t b_ld, const float* b_scales, const void* bias, int activation, void* c, size_t c_ld,
                       void* workspace, size_t workspace_bytes, void* stream) {
    const int out = out_format(dtype);
    if (out < 0) return kNotImplemented;
    if (activation != DLF_B200_ACT_NONE && activation != DLF_B200_ACT_RELU) return kInvalidValue;
    if (m == 0 || n == 0 || k == 0 || m > INT_MAX - 256 || n > INT_MAX - 256 || k > kInt8MaxDepth) return kInvalidDimension;
    if (a_ld < k) return kInvalidLeadDimA;
    if (b_ld < k) return kInvalidLeadDimB;
    if (c_ld < n) return kInvalidLeadDimC;
    if (a == nullptr || a_scales == nullptr) return kInvalidMatrixA;
    if (b == nullptr || b_scales == nullptr) return kInvalidMatrixB;
    if (c == nullptr) return kInvalidMatrixC;
    const size_t need = int8_copy_bytes(m, n, k, a, a_ld, b, b_ld);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return kInsufficientMemoryTemp;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    StreamDevice guard(s);
    if (guard.rc != kSuccess) return guard.rc;
    OperatorDevice dev;
    int rc = operator_device(&dev);
    if (rc != kSuccess) return rc;
    int max_pairs = 0;
    rc = int8_device(dev, &max_pairs);
    if (rc != kSuccess) return rc;
    clear_stale_error();
    Int8Problem q{out, static_cast<long long>(m), static_cast<long long>(n), static_cast<long long>(k), a, static_cast<long long>(a_ld), a_scales,
                  b, static_cast<long long>(b_ld), b_scales, static_cast<const char*>(bias), activation == DLF_B200_ACT_RELU ? 1 : 0,
                  static_cast<char*>(c), static_cast<long long>(c_ld)};
    if (need > 0) {
        rc = int8_copy(dev, q, static_cast<char*>(workspace), s);
        if (rc != kSuccess) return rc;
    }
    if (q.M <= 64) return int8_tile_launch<true>(dev, q, s);
    // pairs where their tiles fill the GPU, else smaller tiles and shared depths
    const long long pair_tiles = ((q.M + 255) / 256) * ((q.N + 255) / 256);
    return 2 * pair_tiles >= max_pairs ? int8_pair_launch(dev, max_pairs, q, s) : int8_tile_launch<false>(dev, q, s);
}

}  // extern "C"
