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

#include "pairs.cuh"
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
    const uint64_t inv2 = ptx::pair_of(inv, inv), up = ptx::pair_of(kMagic, kMagic), down = ptx::pair_of(-kMagic, -kMagic);
    const uint64_t minus = ptx::pair_of(-1.0f, -1.0f);
    uint32_t m[8];
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t t = ptx::mul_pair(ptx::pair_of(p.value(i), p.value(i + 1)), inv2);
        const uint64_t r = ptx::add_pair(t, up);
        float a, b;
        ptx::of_pair(r, a, b);
        m[i] = __float_as_uint(a);
        m[i + 1] = __float_as_uint(b);
        ptx::of_pair(ptx::fma_pair(ptx::add_pair(r, down), minus, t), a, b);
        off = fmaxf(off, fabsf(a));
        off = fmaxf(off, fabsf(b));
    }
    if (off > 0.5f - 0x1p-15f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = static_cast<uint32_t>(quantize_one(p.value(i), s, inv));
    }
    uint2 o;
    o.x = __byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410);
    o.y = __byte_perm(__byte_perm(m[4], m[5], 0x0040), __byte_perm(m[6], m[7], 0x0040), 0x5410);
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
    const int cols = live ? static_cast<int>(p.cols) : 0;
    const int head = min(static_cast<int>(((16u - (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x)) & 15u)) & 15u) / sizeof(T)), cols);
    const int pieces = (cols - head) / 8;
    const int per_warp = (pieces + WARPS * 32 - 1) / (WARPS * 32) * 32;  // (lane l of step j: piece part * per_warp + 32 j + l)
    const int first = min(part * per_warp, pieces), last = min(first + per_warp, pieces), count = last - first;
    const int tail = cols - head - pieces * 8;
    // the odd values are the first warp's: lanes 0-7 the head, 8-15 the tail
    const bool odd = part == 0 && ((lane < 8 && lane < head) || (lane >= 8 && lane - 8 < tail));
    const int odd_at = lane < 8 ? lane : head + pieces * 8 + (lane - 8);
    const T* from = x + head + (first + lane) * 8ll;
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
            if (32 * j + lane < count) held[j].load(from + 256 * j);
            else held[j].clear();
        }
#pragma unroll
        for (int j = 0; j < PIECES; ++j) m = max(m, held[j].largest());
    } else {
        for (int j = 0; j + lane < count; j += 32) {
            held[0].load(from + 8ll * j);
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
    if (count <= 0) return;

    // Piece i makes bytes q[head + 8 i ..]. `shift` of them belong to the aligned eight bytes before the boundary inside
    // the piece (shift = 0: the piece is aligned as it is), the rest to those behind it, with `shift` bytes of the next piece.
    signed char* to = q + head + (first + lane) * 8ll;
    const int shift = static_cast<int>((8u - (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to)) & 7u)) & 7u);
    const bool word = (shift & 4) != 0;
    const uint32_t bits = 8u * (shift & 3);
    uint2 carry = make_uint2(0u, 0u);  // lane 0: the last piece of the step before
    auto put = [&](int j, const QuantizePiece<T>& piece) {  // step of pieces j + lane
        const bool valid = j + lane < count;
        const uint2 v = finite ? quantize_piece(piece, s, inv) : make_uint2(0u, 0u);
        signed char* at = to + 8ll * j;
        if (shift == 0) {
            if (valid) *reinterpret_cast<uint2*>(at) = v;
            return;
        }
        uint2 u;  // the piece before this one
        u.x = __shfl_sync(0xffffffffu, v.x, (lane + 31) & 31);
        u.y = __shfl_sync(0xffffffffu, v.y, (lane + 31) & 31);
        if (lane == 0) {
            const uint2 now = u;
            u = carry;
            carry = now;
        }
        if (!valid) return;
        // the aligned eight bytes that end `shift` bytes into this piece
        if (j + lane == 0) {
            quantize_store_bytes(at, v, 0, shift);
        } else {
            const uint32_t w0 = word ? u.y : u.x, w1 = word ? v.x : u.y, w2 = word ? v.y : v.x;
            *reinterpret_cast<uint2*>(at + shift - 8) = make_uint2(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits));
        }
        if (j + lane == count - 1) quantize_store_bytes(at, v, shift, 8);
    };
    if constexpr (PIECES > 0) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
            if (32 * j < count) put(32 * j, held[j]);
    } else {
        for (int j = 0; j < count; j += 32) {
            if (j + lane < count) held[0].load(from + 8ll * j);
            put(j, held[0]);
        }
    }
}

}  // namespace dlfb200
