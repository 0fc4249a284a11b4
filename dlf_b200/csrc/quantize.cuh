// Rows of floating-point values to 8-bit integers, one scale for each row:
//
//     s_i  = max(rn32(max_j |x_ij| / 127), 2^-126)        (a row with an infinity or a NaN: s_i = NaN, q_ij = 0)
//     q_ij = the whole number nearest to x_ij / s_i, the even one of two equally near
//
// The quotient is the exact one. t = x * rn(1/s) is off by less than 2^-15 (|t| <= 127, two roundings), so the whole
// number nearest to t is q unless t lies that close to the middle between two; then the sign of
// x - (q + 1/2) s decides, which one fused multiply-add gives exactly (quantize_exactly).
//
// HBM-bound: a row is read once and kept in registers between the search for its largest value and the rounding.
// Rows may start anywhere: loads are aligned 16-byte pieces of x with the values before the first and after the last
// piece read one by one; the eight bytes a lane makes of its piece are shifted into the aligned eight bytes of q by one
// exchange with the lane before it (a warp's pieces are consecutive, so only its first and last bytes are stored singly).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace dlfb200 {

struct QuantizeParams {
    const char* x;
    long long x_ld;  // elements
    signed char* q;
    long long q_ld;
    float* scales;
    long long rows;
    long long cols;
};

template <typename T>
__device__ __forceinline__ float quantize_load(const T* p) {
    if constexpr (sizeof(T) == 4) return *p;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(*p);
    else return __bfloat162float(*p);
}

// eight values of x as they lie in memory
template <typename T>
struct QuantizePiece {
    uint32_t w[2 * sizeof(T)];

    __device__ __forceinline__ void load(const T* p) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        if constexpr (sizeof(T) == 4) {
            const uint4 b = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
            w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) w[i] = 0u;
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = *reinterpret_cast<const __half2*>(&w[i >> 1]);
            return (i & 1) ? __high2float(h) : __low2float(h);
        } else {
            return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
        }
    }
    // the largest magnitude as a bit pattern: those of non-negative floats order like whole numbers, with NaN above
    // infinity, so nothing is lost on the way
    __device__ __forceinline__ uint32_t largest() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t m = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
            return m;
        } else {
            uint32_t m = 0u;  // two 16-bit patterns
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            return max(m & 0xffffu, m >> 16);
        }
    }
};

template <typename T>
__device__ __forceinline__ uint32_t quantize_magnitude(T v) {
    if constexpr (sizeof(T) == 4) return __float_as_uint(v) & 0x7fffffffu;
    else return static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(&v)) & 0x7fffu;
}
template <typename T>
__device__ __forceinline__ float quantize_pattern_value(uint32_t m) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(m);
    } else {
        const unsigned short b = static_cast<unsigned short>(m);
        return quantize_load(reinterpret_cast<const T*>(&b));
    }
}

// q for a t = x * rn(1/s) next to the middle of two whole numbers. r = x - q s is exact: near such a middle x is a
// multiple of an ulp of s and |r| < s, but for |x| just under s / 2 with q = +-1, where r may round to -s / 2, which is
// decided like the value below it (q = 0 in both cases).
__device__ __forceinline__ int quantize_exactly(float x, float s, float t) {
    float q = rintf(t);
    const float r = fmaf(-q, s, x), h = 0.5f * s;
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (r > h || (r == h && odd)) q += 1.0f;
    else if (r < -h || (r == -h && odd)) q -= 1.0f;
    return static_cast<int>(q);
}

__device__ __forceinline__ int quantize_one(float x, float s, float inv) {
    const float t = x * inv;
    const float d = t - rintf(t);
    return fabsf(d) > 0.5f - 0x1p-15f ? quantize_exactly(x, s, t) : static_cast<int>(rintf(t));
}

template <typename T>
__device__ __forceinline__ uint2 quantize_piece(const QuantizePiece<T>& p, float s, float inv) {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: the sum's low bits are the rounded value
    float m[8], off = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = p.value(i) * inv;
        m[i] = t + kMagic;
        off = fmaxf(off, fabsf(t - (m[i] - kMagic)));
    }
    if (off > 0.5f - 0x1p-15f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = kMagic + static_cast<float>(quantize_one(p.value(i), s, inv));
    }
    uint2 o;
    o.x = __byte_perm(__byte_perm(__float_as_uint(m[0]), __float_as_uint(m[1]), 0x0040),
                      __byte_perm(__float_as_uint(m[2]), __float_as_uint(m[3]), 0x0040), 0x5410);
    o.y = __byte_perm(__byte_perm(__float_as_uint(m[4]), __float_as_uint(m[5]), 0x0040),
                      __byte_perm(__float_as_uint(m[6]), __float_as_uint(m[7]), 0x0040), 0x5410);
    return o;
}

// bytes [from, to) of eight
__device__ __forceinline__ void quantize_store_bytes(signed char* at, uint2 v, int from, int to) {
    const unsigned long long w = (static_cast<unsigned long long>(v.y) << 32) | v.x;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i >= from && i < to) at[i] = static_cast<signed char>(w >> (8 * i));
}

// A row for every WARPS warps (kQuantizeThreads / 32 / WARPS rows a block); each warp takes consecutive pieces, PIECES a lane at
// most, held in registers. PIECES = 0: rows of any length, read twice.
constexpr int kQuantizeThreads = 256;
template <typename T, int WARPS, int PIECES>
__global__ void __launch_bounds__(kQuantizeThreads) quantize_rows_kernel(const QuantizeParams p) {
    constexpr int kRows = kQuantizeThreads / 32 / WARPS;
    __shared__ uint32_t largest_of[kQuantizeThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = warp % WARPS;
    const long long row = static_cast<long long>(blockIdx.x) * kRows + warp / WARPS;
    const bool live = row < p.rows;
    const T* x = reinterpret_cast<const T*>(p.x) + (live ? row : 0) * p.x_ld;
    signed char* q = p.q + (live ? row : 0) * p.q_ld;
    ptx::launch_dependents();
    ptx::wait_for_dependencies();

    // head values before the first 16-byte boundary, whole pieces of eight, tail values
    const long long cols = live ? p.cols : 0;
    const int head = static_cast<int>(min(static_cast<long long>(((16u - (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x)) & 15u)) & 15u) / sizeof(T)), cols));
    const long long pieces = (cols - head) / 8;
    const long long per_warp = (pieces + WARPS * 32 - 1) / (WARPS * 32) * 32;  // (lane l of step j: piece part * per_warp + 32 j + l)
    const long long first = min(part * per_warp, pieces), last = min(first + per_warp, pieces);
    const int tail = static_cast<int>(cols - head - pieces * 8);
    // the odd values are the first warp's: lanes 0-7 the head, 8-15 the tail
    const bool odd = part == 0 && ((lane < 8 && lane < head) || (lane >= 8 && lane - 8 < tail));
    const long long odd_at = lane < 8 ? lane : head + pieces * 8 + (lane - 8);
    uint32_t m = 0u;
    float odd_x = 0.0f;
    if (odd) {
        const T v = x[odd_at];
        m = quantize_magnitude(v);
        odd_x = quantize_load(&v);
    }
    QuantizePiece<T> held[PIECES > 0 ? PIECES : 1];
    if constexpr (PIECES > 0) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const long long i = first + 32 * j + lane;
            if (i < last) held[j].load(x + head + i * 8);
            else held[j].clear();
        }
#pragma unroll
        for (int j = 0; j < PIECES; ++j) m = max(m, held[j].largest());
    } else {
        for (long long i = first + lane; i < last; i += 32) {
            held[0].load(x + head + i * 8);
            m = max(m, held[0].largest());
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (WARPS > 1) {
        if (lane == 0) largest_of[warp] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = max(m, largest_of[warp / WARPS * WARPS + w]);
    }
    if (!live) return;
    const float amax = quantize_pattern_value<T>(m);
    const bool finite = amax <= 3.402823466e38f;
    const float s = finite ? fmaxf(__fdiv_rn(amax, 127.0f), 0x1p-126f) : __uint_as_float(0x7fc00000u);
    const float inv = __fdiv_rn(1.0f, s);
    if (part == 0 && lane == 0) p.scales[row] = s;
    if (odd) q[odd_at] = finite ? static_cast<signed char>(quantize_one(odd_x, s, inv)) : static_cast<signed char>(0);

    // Piece i makes bytes q[head + 8 i ..]. `shift` of them belong to the aligned eight bytes before the boundary inside
    // the piece (shift = 0: the piece is aligned as it is).
    const uint32_t lead = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(q + head)) & 7u;
    const int shift = static_cast<int>((8u - lead) & 7u);
    uint2 before = make_uint2(0u, 0u);  // the last piece of the step before
    auto put = [&](long long i0, const QuantizePiece<T>& piece) {
        const long long i = i0 + lane;
        const bool valid = i < last;
        uint2 v = finite ? quantize_piece(piece, s, inv) : make_uint2(0u, 0u);
        signed char* at = q + head + i * 8;
        if (shift == 0) {
            if (valid) *reinterpret_cast<uint2*>(at) = v;
            return;
        }
        uint2 u;  // the piece before this one
        u.x = __shfl_up_sync(0xffffffffu, v.x, 1);
        u.y = __shfl_up_sync(0xffffffffu, v.y, 1);
        if (lane == 0) u = before;
        before.x = __shfl_sync(0xffffffffu, v.x, 31);
        before.y = __shfl_sync(0xffffffffu, v.y, 31);
        if (!valid) return;
        // the aligned eight bytes that end `shift` bytes into this piece
        if (i == first) {
            quantize_store_bytes(at, v, 0, shift);
        } else {
            const unsigned long long lo = (static_cast<unsigned long long>(u.y) << 32) | u.x, hi = (static_cast<unsigned long long>(v.y) << 32) | v.x;
            const unsigned long long w = (lo >> (8 * shift)) | (hi << (64 - 8 * shift));
            *reinterpret_cast<unsigned long long*>(at + shift - 8) = w;
        }
        if (i == last - 1) quantize_store_bytes(at, v, shift, 8);
    };
    if constexpr (PIECES > 0) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
            if (first + 32 * j < last) put(first + 32 * j, held[j]);
    } else {
        for (long long i0 = first; i0 < last; i0 += 32) {
            if (i0 + lane < last) held[0].load(x + head + (i0 + lane) * 8);
            put(i0, held[0]);
        }
    }
}

}  // namespace dlfb200
