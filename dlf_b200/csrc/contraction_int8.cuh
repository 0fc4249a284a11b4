// Products of 8-bit integers with a scale for each row of A (token) and each row of B (output channel):
//
//     D[i*ldd + j] = act((sum_k A[i][k] B[j][k]) * sb[j] * sa[i] + bias[j])
//
// The sums are 32-bit integers in tensor memory (tcgen05.mma.kind::i8), so they are exact (K <= 131071) and may be split
// and added in any order. The scale of the channel is applied before that of the token: weights have tame scales, so the
// intermediate value overflows no earlier than the result does.
//
// int8_tile_kernel: one tile of 128 x BN per cluster of S CTAs that share its k-blocks; see below.
// int8_pair_kernel: persistent, tiles of 256 x 256 that two CTAs share (cta_group::2).
//
// Operand tiles are K-major with 128-byte lines (128 k-values) in the 128-byte-swizzled canonical layout, by TMA; lines past
// an operand's end and k-values past K arrive as zeros.
#pragma once
#include "contraction.cuh"
#include "contraction_split.cuh"
#include "dependents.cuh"

namespace dlfb200 {

namespace ptx {
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "}"
        :
        : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "}"
        :
        : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// kind::i8, both operands signed and K-major, 32-bit integer accumulator: bits 4-5 D format (2 = s32), bits 7-9 and 10-12 A and B
// format (1 = s8), the sizes as in make_idesc
__host__ __device__ __forceinline__ uint32_t make_idesc_i8(uint32_t m, uint32_t n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
}  // namespace ptx

struct Int8Params {
    int M, N, K;            // rows of A (tokens), rows of B (channels), depth
    int BN, stages, S;      // tile columns, ring stages, CTAs that share a tile's k-blocks
    int tiles_l, tiles_c;   // tiles along the lanes and along the columns
    const float* sa;
    const float* sb;
    const char* bias;
    int relu;
    char* d;
    long long ldd;
    int vec;                // lines of D take 16-byte stores
    int* status;
    long long wait_limit;
    int withhold;           // test aid: the issuer leaves out the commit that ends the tile
};

__device__ __forceinline__ int ld_shared_s32(uint32_t addr) {
    int v;
    asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

constexpr int kInt8Threads = 256;
constexpr int kInt8MaxStages = 12;
constexpr int int8_tile_part_bytes(int bn) { return kBM * (bn + 4) * 4; }
constexpr int int8_tile_smem(int bn, int stages) {
    return 1024 + (stages * (kBM + bn) * 128 > int8_tile_part_bytes(bn) ? stages * (kBM + bn) * 128 : int8_tile_part_bytes(bn));
}

__device__ __forceinline__ float int8_scaled(int acc, float sb, float sa, float bias, int relu) {
    const float v = fmaf(static_cast<float>(acc) * sb, sa, bias);
    return relu && v < 0.0f ? 0.0f : v;  // (a NaN stays one)
}

// One tile per cluster; the S partial tiles meet in distributed shared memory, where CTA r adds its share of them. CHANNELS: the
// lanes are output channels and the columns tokens (few tokens: the weights are what is read, and 128 lanes of them use the
// tensor core's fixed 128 rows); else the lanes are tokens.
// Roles as in contraction_split_kernel: warps 0-3 read the accumulator, 4 TMA producer, 5 UMMA issuer and TMEM owner, all write.
template <int OUT, bool CHANNELS>
__global__ void __launch_bounds__(kInt8Threads)
    int8_tile_kernel(const __grid_constant__ Int8Params p, const __grid_constant__ CUtensorMap tmL,
                     const __grid_constant__ CUtensorMap tmC) {
    constexpr int BK = 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kInt8MaxStages];
    __shared__ __align__(8) uint64_t empty_bar[kInt8MaxStages];
    __shared__ __align__(8) uint64_t done_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ float token_scale[CHANNELS ? 1 : kBM];

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const int S = p.S, BN = p.BN;
    const int rank = S > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const uint32_t smem0 = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t stage_bytes = static_cast<uint32_t>(kBM + BN) * 128u;
    const int num_kb = (p.K + BK - 1) / BK;
    const int kb0 = rank * num_kb / S, kb1 = (rank + 1) * num_kb / S;
    const int tile = blockIdx.x / S;
    const int tc = tile / p.tiles_l, tl = tile - tc * p.tiles_l;
    const int l0 = tl * kBM, c0 = tc * BN;
    const uint32_t tmem_cols = BN <= 32 ? 32u : static_cast<uint32_t>(BN);  // (BN: a power of two)

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < p.stages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1u);
            ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1u);
        }
        ptx::mbar_init(ptx::smem_u32(&done_bar), 1u);
        ptx::fence_mbar_init();
    }
    if (warp == 5) {
        __syncwarp();
        ptx::tmem_alloc_then_dependents(ptx::smem_u32(&tmem_slot), tmem_cols);
    }
    if (warp == 4 && lane == 0) {
        ptx::tma_prefetch_desc(&tmL);
        ptx::tma_prefetch_desc(&tmC);
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
    volatile int* abort_p = &abort_flag;
    const long long wait_limit = p.wait_limit;
    // The first of the weights, as many as the ring holds, on their way into L2 while the kernel before this one (the quantisation of the
    // tokens) finishes. All of them would be more than L2 holds and get in the way of the loads themselves: 16 x 16384 x 16384 read
    // 338 MB for 268 in 58.5 us, so 46.5 (none asked for: 48.2); 16 x 4096 x 4096 9.2 us either way (none: 9.7).
    if (CHANNELS && warp == 4 && ptx::elect_one())
        for (int kb = kb0; kb < min(kb1, kb0 + p.stages); ++kb) ptx::tma_prefetch_3d(&tmL, kb * BK, l0, 0);
    __syncwarp();
    ptx::wait_for_dependencies();

    // The scale and the bias of the channel that this thread writes, asked for beside the products; the tokens' scales come by way of
    // shared memory (both asked for behind the products: fp32 1111 x 1537 x 784 9.8 us, so 9.1; where CTAs share a depth a thread writes
    // four channels, and that the other way round was 0.3 us slower).
    float chan_scale = 0.0f, chan_bias = 0.0f;
    if (CHANNELS || S == 1) {
        const int j = CHANNELS ? l0 + (rank * (min(BN, p.M - c0) * kBM / 32) / S * 32 + static_cast<int>(threadIdx.x)) % kBM
                               : c0 + static_cast<int>(threadIdx.x) % BN;
        if (j < p.N) {
            chan_scale = p.sb[j];
            if (p.bias != nullptr) chan_bias = out_load<OUT>(p.bias + static_cast<long long>(j) * (OUT == OUT_F32 ? 4 : 2));
        }
        if (!CHANNELS && warp >= 6)
            for (int r = static_cast<int>(threadIdx.x) - 192; r < kBM; r += 64) token_scale[r] = p.sa[min(l0 + r, p.M - 1)];
    }

    if (warp == 4) {
        // ------------------------------------------------------------ TMA producer
        const bool leader = ptx::elect_one();
        uint32_t s = 0, ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(ptx::smem_u32(&empty_bar[s]), ph ^ 1u, abort_p, wait_limit))) break;
            const uint32_t bar = ptx::smem_u32(&full_bar[s]);
            const uint32_t sL = smem0 + s * stage_bytes;
            if (leader) {
                ptx::mbar_arrive_expect_tx(bar, stage_bytes);
                ptx::tma_load_3d(sL, &tmL, bar, kb * BK, l0, 0);
                ptx::tma_load_3d(sL + kBM * 128, &tmC, bar, kb * BK, c0, 0);
            }
            __syncwarp();
            if (++s == static_cast<uint32_t>(p.stages)) {
                s = 0;
                ph ^= 1u;
            }
        }
    } else if (warp == 5) {
        // ------------------------------------------------------------ UMMA issuer
        const uint32_t idesc = ptx::make_idesc_i8(kBM, static_cast<uint32_t>(BN));
        const uint64_t da0 = ptx::make_smem_desc(smem0, 16u, 1024u, 2u);
        const uint64_t db0 = ptx::make_smem_desc(smem0 + kBM * 128, 16u, 1024u, 2u);
        uint32_t s = 0, ph = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(ptx::smem_u32(&full_bar[s]), ph, abort_p, wait_limit))) {
                ok = false;
                break;
            }
            ptx::tc_fence_after();
            const uint32_t at = (s * stage_bytes) >> 4;
            if (ptx::elect_one()) {
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    ptx::umma_i8(tmem, da0 + (at + ks * 2), db0 + (at + ks * 2), idesc, (kb > kb0 || ks > 0) ? 1u : 0u);
                ptx::umma_commit(ptx::smem_u32(&empty_bar[s]));
            }
            __syncwarp();
            if (++s == static_cast<uint32_t>(p.stages)) {
                s = 0;
                ph ^= 1u;
            }
        }
        if (ok && !p.withhold && ptx::elect_one()) ptx::umma_commit(ptx::smem_u32(&done_bar));
        __syncwarp();
    } else if (warp < 4) {
        // ------------------------------------------------------------ accumulator -> partial tile
        // (the operand ring is free by then: every copy into it has been consumed). Lines of BN + 4 (tokens in the lanes, read
        // along the columns, four at a time) or BN + 1 (read along the lanes) integers: neither has bank conflicts.
        if (__all_sync(0xffffffffu, ptx::mbar_wait_bounded(ptx::smem_u32(&done_bar), 0u, abort_p, wait_limit))) {
            ptx::tc_fence_after();
            const uint32_t ld = static_cast<uint32_t>(CHANNELS ? BN + 1 : BN + 4) * 4u;
            const uint32_t row = smem0 + static_cast<uint32_t>(warp * 32 + lane) * ld;
#pragma unroll 1
            for (int h = 0; h < BN; h += 16) {
                uint32_t v[16];
                ptx::tmem_ld_32x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + h, v);
                ptx::tmem_ld_wait();
                if constexpr (CHANNELS) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(row + (h + j) * 4), "r"(v[j]) : "memory");
                } else {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) st_shared_v4(row + (h + j) * 4, make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]));
                }
            }
            ptx::tc_fence_before();
        }
    }
    __syncthreads();
    if (abort_flag) {
        // copies and UMMAs still in flight get time to land before shared and tensor memory are released
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        if (threadIdx.x == 0) atomicOr(p.status, DEV_STATUS_WAIT_TIMEOUT);
    }
    if (S > 1) ptx::cluster_sync();
    int gave_up = abort_flag;
    if (S > 1) gave_up = lane < S ? ptx::ld_cluster_s32(ptx::map_to_cta(ptx::smem_u32(&abort_flag), lane)) : 0;
    if (!__any_sync(0xffffffffu, gave_up != 0)) {
        constexpr int OES = OUT == OUT_F32 ? 4 : 2;
        if constexpr (CHANNELS) {
            // values in the order token, channel: a warp writes 32 channels of one token
            const int live = min(BN, p.M - c0) * kBM;
            const int i0 = rank * (live / 32) / S * 32, i1 = (rank + 1) * (live / 32) / S * 32;
            const int c = (i0 + static_cast<int>(threadIdx.x)) % kBM, j = l0 + c;  // (a thread's channel stays the same)
            for (int id = i0 + static_cast<int>(threadIdx.x); id < i1 && j < p.N; id += kInt8Threads) {
                const int t = id / kBM;
                const uint32_t at = smem0 + static_cast<uint32_t>((c * (BN + 1) + t) * 4);
                int v[kSplitMaxCtas];
#pragma unroll
                for (int k = 0; k < kSplitMaxCtas; ++k)
                    if (k < S) v[k] = ptx::ld_cluster_s32(S > 1 ? ptx::map_to_cta(at, k) : at);
                int acc = 0;
#pragma unroll
                for (int k = 0; k < kSplitMaxCtas; ++k)
                    if (k < S) acc += v[k];
                const int i = c0 + t;
                out_store<OUT>(p.d + (static_cast<long long>(i) * p.ldd + j) * OES, int8_scaled(acc, chan_scale, p.sa[i], chan_bias, p.relu));
            }
        } else if (S > 1) {
            // four columns a thread, always the same ones: what costs is the loads from other SMs, so few of them
            const int r0 = rank * kBM / S, r1 = (rank + 1) * kBM / S, groups = BN / 4;
            const int c = static_cast<int>(threadIdx.x) % groups * 4, j = c0 + c;
            float sb[4], bias[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sb[e] = j + e < p.N ? p.sb[j + e] : 0.0f;
                bias[e] = p.bias != nullptr && j + e < p.N ? out_load<OUT>(p.bias + static_cast<long long>(j + e) * OES) : 0.0f;
            }
#pragma unroll 2
            for (int r = r0 + static_cast<int>(threadIdx.x) / groups; r < r1; r += kInt8Threads / groups) {
                const int i = l0 + r;
                if (i >= p.M || j >= p.N) break;
                const uint32_t at = smem0 + static_cast<uint32_t>((r * (BN + 4) + c) * 4);
                float4 v[kSplitMaxCtas];
#pragma unroll
                for (int k = 0; k < kSplitMaxCtas; ++k)
                    if (k < S) v[k] = ptx::ld_cluster_v4(ptx::map_to_cta(at, k));
                int acc[4] = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < kSplitMaxCtas; ++k) {
                    if (k < S) {
                        acc[0] += __float_as_int(v[k].x);
                        acc[1] += __float_as_int(v[k].y);
                        acc[2] += __float_as_int(v[k].z);
                        acc[3] += __float_as_int(v[k].w);
                    }
                }
                const float sa = p.sa[i];
                char* dst = p.d + (static_cast<long long>(i) * p.ldd + j) * OES;
                __align__(16) char o[4 * OES];
#pragma unroll
                for (int e = 0; e < 4; ++e) out_store<OUT>(o + e * OES, int8_scaled(acc[e], sb[e], sa, bias[e], p.relu));
                if (p.vec && j + 4 <= p.N) {
                    if constexpr (OES == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(o);
                    else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (j + e < p.N) {
                            if constexpr (OES == 4) reinterpret_cast<uint32_t*>(dst)[e] = reinterpret_cast<const uint32_t*>(o)[e];
                            else reinterpret_cast<unsigned short*>(dst)[e] = reinterpret_cast<const unsigned short*>(o)[e];
                        }
                }
            }
        } else {
            // a column a thread, so that a warp writes neighbours wherever the lines of D start, and its scale and bias are read once
            // (fp32 1111 x 1537 x 784 11.1 us, four columns a thread 14.4; 1111 x 1536 x 784 11.1 and 12.0)
            const int c = static_cast<int>(threadIdx.x) % BN, j = c0 + c;
            const int step = kInt8Threads / BN;
            for (int r = static_cast<int>(threadIdx.x) / BN; r < kBM && l0 + r < p.M && j < p.N; r += 8 * step) {
                // eight rows at a time: their loads are all asked for before the first value is used
                int acc[8];
                float sa[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const int rx = min(r + x * step, kBM - 1);
                    sa[x] = token_scale[rx];
                    acc[x] = ld_shared_s32(smem0 + static_cast<uint32_t>((rx * (BN + 4) + c) * 4));
                }
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const int i = l0 + r + x * step;
                    if (r + x * step < kBM && i < p.M)
                        out_store<OUT>(p.d + (static_cast<long long>(i) * p.ldd + j) * OES, int8_scaled(acc[x], chan_scale, sa[x], chan_bias, p.relu));
                }
            }
        }
    }
    if (S > 1) ptx::cluster_sync();  // no CTA leaves while another still reads its partial tile
    if (warp == 5) {
        __syncwarp();
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, tmem_cols);
    }
}

// Persistent: pairs of CTAs walk through tiles of 256 x 256 (tokens x channels). Each CTA of a pair stages its 128 rows of A and
// half the rows of B, one issuer drives both tensor cores (cta_group::2), which halves what B costs in shared-memory reads and
// fills; the two accumulators of 256 columns take all of tensor memory, so a tile's epilogue runs beside the next
// tile's products. Bound by the tensor core (8192^3: 334 us in a short run) and, in a row, by the
// power cap (381 us, 1.30 GHz at 993 W) from a depth of about 512 on, below by the epilogue's conversions.
// Roles: warps 0-3 and 6-9 epilogue (quadrant = warp % 4, half of the columns each), 4 UMMA issuer and TMEM owner, 5 TMA producer.
constexpr int kInt8PairThreads = 320;
constexpr int kInt8PairStages = 6;
constexpr int kInt8PairBN = 256;
constexpr int kInt8PairStageBytes = 2 * kBM * 128;
constexpr int kInt8PairSmem = 1024 + kInt8PairStages * kInt8PairStageBytes + 8 * 4096;

__device__ __forceinline__ void int8_pair_tile(const Int8Params& p, int t, int& m0, int& n0) {
    const int group = kGroupM * p.tiles_c, gi = t / group, r = t - gi * group;
    const int gm = min(p.tiles_l - gi * kGroupM, kGroupM), cq = r / gm;
    m0 = (gi * kGroupM + r - cq * gm) * 2 * kBM;
    n0 = cq * kInt8PairBN;
}

template <int OUT>
__global__ void __launch_bounds__(kInt8PairThreads, 1)
    int8_pair_kernel(const __grid_constant__ Int8Params p, const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmD) {
    constexpr int BK = 128, OES = OUT == OUT_F32 ? 4 : 2;
    constexpr int COLS = 128 / OES;  // columns of a staging block: lines of 128 bytes
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kInt8PairStages], empty_bar[kInt8PairStages], tfull_bar[2], tempty_bar[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_ctarank();
    const uint32_t smem0 = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const int num_kb = (p.K + BK - 1) / BK;
    const int tiles = p.tiles_l * p.tiles_c, tile0 = blockIdx.x / 2, step = gridDim.x / 2;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < kInt8PairStages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1u);
            ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1u);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(ptx::smem_u32(&tfull_bar[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&tempty_bar[i]), 16u);  // the epilogue warps of both CTAs, on rank 0's barrier
        }
        ptx::fence_mbar_init();
    }
    if (warp == 4) {
        __syncwarp();
        ptx::tmem_alloc_pair_then_dependents(ptx::smem_u32(&tmem_slot), 512u);
    }
    if (warp == 5 && lane == 0) {
        ptx::tma_prefetch_desc(&tmA);
        ptx::tma_prefetch_desc(&tmB);
        ptx::tma_prefetch_desc(&tmD);
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();  // the peer's barriers exist before anything remote happens
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
    volatile int* abort_p = &abort_flag;
    const long long limit = p.wait_limit;
    ptx::wait_for_dependencies();
    auto wait = [&](uint64_t& bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, ptx::mbar_wait_bounded(ptx::smem_u32(&bar), parity, abort_p, limit));
    };

    if (warp == 5) {
        // ------------------------------------------------------------ TMA producer
        const bool leader = ptx::elect_one();
        uint32_t s = 0, ph = 0;
        bool ok = true;
        for (int t = tile0; ok && t < tiles; t += step) {
            int m0, n0;
            int8_pair_tile(p, t, m0, n0);
            m0 += static_cast<int>(rank) * kBM;
            n0 += static_cast<int>(rank) * kBM;  // this CTA's share of B's rows
            for (int kb = 0; kb < num_kb; ++kb) {
                ok = wait(empty_bar[s], ph ^ 1u);
                if (!ok) break;
                // both CTAs' copies are counted on rank 0's barrier, which rank 0 arms with the bytes of the two together
                const uint32_t bar = ptx::map_to_cta(ptx::smem_u32(&full_bar[s]), 0u);
                const uint32_t sA = smem0 + s * kInt8PairStageBytes;
                if (leader) {
                    if (rank == 0) ptx::mbar_arrive_expect_tx(ptx::smem_u32(&full_bar[s]), 2u * kInt8PairStageBytes);
                    ptx::tma_load_3d_pair(sA, &tmA, bar, kb * BK, m0, 0);
                    ptx::tma_load_3d_pair(sA + kBM * 128, &tmB, bar, kb * BK, n0, 0);
                }
                __syncwarp();
                if (++s == kInt8PairStages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
    } else if (warp == 4) {
        // ------------------------------------------------------------ UMMA issuer (rank 0's)
        if (rank == 0) {
            const uint32_t idesc = ptx::make_idesc_i8(2 * kBM, kInt8PairBN);
            const uint64_t da0 = ptx::make_smem_desc(smem0, 16u, 1024u, 2u);
            const uint64_t db0 = ptx::make_smem_desc(smem0 + kBM * 128, 16u, 1024u, 2u);
            uint32_t s = 0, ph = 0, it = 0;
            bool ok = true;
            for (int t = tile0; ok && t < tiles; t += step, ++it) {
                const uint32_t buf = it & 1u;
                ok = wait(tempty_bar[buf], ((it >> 1) & 1u) ^ 1u);
                if (!ok) break;
                ptx::tc_fence_after();
                for (int kb = 0; kb < num_kb; ++kb) {
                    ok = wait(full_bar[s], ph);
                    if (!ok) break;
                    ptx::tc_fence_after();
                    const uint32_t at = (s * kInt8PairStageBytes) >> 4;
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            ptx::umma_i8_pair(tmem + buf * kInt8PairBN, da0 + (at + ks * 2), db0 + (at + ks * 2), idesc, (kb > 0 || ks > 0) ? 1u : 0u);
                        ptx::umma_commit_pair(ptx::smem_u32(&empty_bar[s]));
                        ptx::umma_commit_pair(ptx::map_to_cta(ptx::smem_u32(&empty_bar[s]), 1u));
                        if (kb + 1 == num_kb) {
                            ptx::umma_commit_pair(ptx::smem_u32(&tfull_bar[buf]));
                            ptx::umma_commit_pair(ptx::map_to_cta(ptx::smem_u32(&tfull_bar[buf]), 1u));
                        }
                    }
                    __syncwarp();
                    if (++s == kInt8PairStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue
        const int q = warp & 3, ewarp = warp < 4 ? warp : warp - 2, half = warp < 4 ? 0 : 1;
        const uint32_t stage = smem0 + kInt8PairStages * kInt8PairStageBytes + ewarp * 4096u;
        const uint32_t line = stage + lane * 128u, sx = static_cast<uint32_t>(lane) & 7u;
        uint32_t it = 0;
        for (int t = tile0; t < tiles; t += step, ++it) {
            int m0, n0;
            int8_pair_tile(p, t, m0, n0);
            const int i0 = m0 + static_cast<int>(rank) * kBM + q * 32;
            const uint32_t buf = it & 1u;
            if (!wait(tfull_bar[buf], (it >> 1) & 1u)) break;
            ptx::tc_fence_after();
            const uint32_t trow = tmem + (static_cast<uint32_t>(q * 32) << 16) + buf * kInt8PairBN;
            const float sa = i0 + lane < p.M ? p.sa[i0 + lane] : 0.0f;
            for (int c0 = half * 128; c0 < half * 128 + 128 && i0 < p.M; c0 += COLS) {
                const int j0 = n0 + c0;
                if (j0 >= p.N) break;
                if (lane == 0) ptx::bulk_wait_group_read<0>();
                __syncwarp();
#pragma unroll
                for (int h = 0; h < COLS / 32; ++h) {
                    uint32_t v[32];
                    ptx::tmem_ld_32x32(trow + c0 + 32 * h, v);
                    ptx::tmem_ld_wait();
                    const int j = j0 + 32 * h + lane;
                    const float sb = j < p.N ? p.sb[j] : 0.0f;
                    const float bias = p.bias != nullptr && j < p.N ? out_load<OUT>(p.bias + static_cast<long long>(j) * OES) : 0.0f;
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        v[x] = __float_as_uint(int8_scaled(static_cast<int>(v[x]), __shfl_sync(0xffffffffu, sb, x), sa, __shfl_sync(0xffffffffu, bias, x), p.relu));
                    constexpr int PER = 16 / OES;  // values of a 16-byte piece
#pragma unroll
                    for (int k = 0; k < 32 / PER; ++k) {
                        __align__(16) char o[16];
#pragma unroll
                        for (int e = 0; e < PER; ++e) out_store<OUT>(o + e * OES, __uint_as_float(v[k * PER + e]));
                        const uint32_t ch = static_cast<uint32_t>(h * (32 / PER) + k);
                        st_shared_v4(line + ((ch ^ sx) << 4), *reinterpret_cast<const uint4*>(o));
                    }
                }
                if (p.vec) {
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::tma_store_3d(&tmD, stage, j0, i0, 0);
                        ptx::bulk_commit_group();
                    }
                } else {
                    // lines of D that the tensor map cannot take: value by value, a line at a time
                    __syncwarp();
                    for (int r = 0; r < 32 && i0 + r < p.M; ++r)
#pragma unroll
                        for (int x = 0; x < COLS; x += 32) {
                            const int col = x + lane;
                            if (j0 + col >= p.N) continue;
                            const uint32_t at = stage + r * 128u + (((static_cast<uint32_t>(col * OES) >> 4) ^ (r & 7u)) << 4) + (col * OES & 15);
                            char* dst = p.d + (static_cast<long long>(i0 + r) * p.ldd + j0 + col) * OES;
                            if constexpr (OES == 4) {
                                uint32_t u;
                                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(u) : "r"(at) : "memory");
                                *reinterpret_cast<uint32_t*>(dst) = u;
                            } else {
                                unsigned short u;
                                asm volatile("ld.shared.b16 %0, [%1];" : "=h"(u) : "r"(at) : "memory");
                                *reinterpret_cast<unsigned short*>(dst) = u;
                            }
                        }
                    __syncwarp();
                }
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_cta(ptx::smem_u32(&tempty_bar[buf]), 0u));
        }
        if (lane == 0) ptx::bulk_wait_group_read<0>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (*abort_p) {
        // copies and UMMAs still in flight get time to land before shared and tensor memory are released
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        if (threadIdx.x == 0) atomicOr(p.status, DEV_STATUS_WAIT_TIMEOUT);
        __syncthreads();
    }
    ptx::cluster_sync();  // the peer may still signal this CTA's barriers until here
    if (warp == 4) {
        __syncwarp();
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem, 512u);
    }
}

// Lines of an operand that start anywhere, copied so that they start on 16-byte boundaries (blockIdx.y: which operand); the bytes
// past a line's end are zero. A thread writes 16 bytes from four aligned words; where the line starts off their boundaries from three and the
// four bytes beside those one by one, so that nothing outside the line is read; the last bytes of a line one by one.
struct Int8Lines {
    const signed char* src[2];
    signed char* dst[2];
    long long src_pitch[2], lines[2];
    int length, dst_pitch;
};
__global__ void __launch_bounds__(256) int8_lines_kernel(const Int8Lines p) {
    const int m = blockIdx.y;
    const unsigned chunks = static_cast<unsigned>(p.dst_pitch / 16);
    const unsigned long long total = static_cast<unsigned long long>(p.lines[m]) * chunks;
    ptx::launch_dependents();
    ptx::wait_for_dependencies();
    // (line by line where the count of pieces passes 32 bits)
    const bool small = total < 0x80000000ull;
    for (unsigned long long id = static_cast<unsigned long long>(blockIdx.x) * blockDim.x + threadIdx.x; id < total; id += static_cast<unsigned long long>(gridDim.x) * blockDim.x) {
        const long long line = small ? static_cast<long long>(static_cast<unsigned>(id) / chunks) : static_cast<long long>(id / chunks);
        const int e0 = static_cast<int>(id - static_cast<unsigned long long>(line) * chunks) * 16;
        const signed char* at = p.src[m] + line * p.src_pitch[m] + e0;
        uint32_t o[4];
        if (e0 + 16 <= p.length) {
            const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at)) & 3u;
            if (off == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = reinterpret_cast<const uint32_t*>(at)[i];
            } else {
                // three words lie between the first and the last of these 16 bytes; the two at the ends need not lie in the line: what
                // is wanted of them is read byte by byte
                uint32_t w[5];
                const uint32_t* a = reinterpret_cast<const uint32_t*>(at - off);
                w[0] = 0u;
                w[4] = 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i >= static_cast<int>(off)) w[0] |= static_cast<uint32_t>(static_cast<uint8_t>(at[i - static_cast<int>(off)])) << (8 * i);
                    if (i < static_cast<int>(off)) w[4] |= static_cast<uint32_t>(static_cast<uint8_t>(at[16 - static_cast<int>(off) + i])) << (8 * i);
                }
#pragma unroll
                for (int i = 1; i < 4; ++i) w[i] = a[i];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(w[i], w[i + 1], 8u * off);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = 0u;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (e0 + i < p.length) o[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(at[i])) << (8 * (i & 3));
        }
        *reinterpret_cast<uint4*>(p.dst[m] + line * p.dst_pitch + e0) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace dlfb200
