// Attention of many query rows over more than 128 keys: two tiles of 128 queries per CTA against tiles of 128 keys, on the tensor cores.
//
//     S = Q K^T,  p = exp2(c (S - m)),  O = sum over key tiles of P V,  y = O / sum p      (c = scale * log2 e)
//
// The difference is taken first (attention_decode.cuh says why) where c m is beyond 2^10; below, the rounding of c m is 2^-14 at most,
// and one fused step for c S - c m saves 3 % (2 x 4096 x up to 8192, 32 heads of 128: 769 us with the difference always, 739 so).
// m is a reference near the running maximum of a row: it is moved (and O and the sum scaled) only when the maximum has grown by
// more than 2^8 since, which exp2's range allows and which makes the pass over O rare. In fp16 p is taken times 2^7, as in
// attention_decode.cuh.
//
// With heads of 128 values (2 x 4096 x 4096, 32 heads: 506 us and 1090 TFLOP/s in a short run, 546 us and 1010 in a long one) the clock is
// what gives way, 1.60 GHz at 990 W under the power cap; but no unit is full - tensor pipe 56 %, special-function unit 56 %, issue
// slots 51 % - and plain products keep 1420 TFLOP/s under the same cap, so it is what this arrangement costs: S with both operands in
// shared memory reads 8 KB in the 64 clocks of a product of 128 x 128 x 16, all that shared memory gives, and each tile of queries reads
// K and V for itself. With heads of 64 latencies and the special-function unit (59 %; tensor pipe 29 %, the clock near its maximum): a
// pair of tiles of 128 x 128 scores costs the tensor core 1024 clocks and exp2, 16 a clock, 2048; it takes 3500.
//
// Tensor memory (512 columns): O of the two tiles (DP columns each), P of the two tiles (16-bit pairs, 64 columns each; the A
// operand of P V, so the scores never touch shared memory), and S: 128 columns for each tile with heads of 64, 128 columns that the tiles
// use in turn with heads of 128. A thread takes its part of S into registers at once, so S is free again for the next product
// while the exponentials are computed (with P in S's place the next S has to wait for P V). P is rounded to the 16-bit type
// once (the tensor core takes both operands of one type, and a second part for the rest, as attention_decode.cuh has it, would be
// half as many products again): an error of half a step of the type for each p, as large as that of the result's own rounding (bf16,
// 4096 x 8192: 2.3e-3 in all, 1.7e-3 from the result's). O and the sums are 32-bit.
//
// Roles: warps 0-15 the softmax - 8 for each tile, a thread for half a query row (64 keys of a tile; the halves exchange their
// maxima and sums through shared memory): with one thread a row (8 warps) heads of 64 and short rows took a tenth longer - 16 and
// 18 issue the products of tile 0 and 1 (each in the order next S, P V; one issuer for both makes each wait for the other's
// softmax), 17 TMA loads, 19 zeroes the value rows of keys that do not count (0 * NaN would be NaN).
// K and V tiles go through one ring in the order of their use: K0, K1, V0, K2, V1, ...
//
// The work is shared out in units of one tile of keys (attention_plan.h; a "head" there is a head and a pair of query tiles): every
// CTA takes the same number, and what is cut leaves O and the sums in 32 bits for attention_tiles_join_kernel. The next segment's loads
// and (heads of 64) first products run beside this one's last. A whole result is staged in the segment's own Q buffer and leaves by
// TMA stores, 32 rows and half a head a warp.
#pragma once
#include <cuda.h>

#include "attention_decode.cuh"
#include "attention_plan.h"
#include "dependents.cuh"
#include "pairs.cuh"
#include "ptx.cuh"

namespace dlfb200 {

namespace ptx {
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        :
        : "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
                 :
                 : "l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem desc]
__device__ __forceinline__ void umma_f16_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}"
        :
        : "r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        :
        : "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
          "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
          "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]),
          "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        :
        : "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
          "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
}  // namespace ptx

struct TilesParams {
    int batch, queries, keys, heads, group, size;
    const int* lengths;         // or null: `keys` each
    const unsigned char* mask;  // (batch, keys) or null
    long long mask_sb;
    int q_pairs, ctas;
    int k_batched, v_batched, q_batched;  // 0: the operand is shared by the batch
    float c;
    char* y;
    long long y_sb, y_st, y_sh;  // elements; for the joining kernel
    float* parts;                // slots of 256 x (size + 2) floats: O, then maximum and sum per row
    int* status;
    long long wait_limit;
    int withhold;  // test aid: the commit that ends a segment is left out
};

constexpr int kTilesThreads = 640;
constexpr int kTileKeys = 128;
constexpr int kTileBlock = 128 * 128;  // bytes of 128 rows x 64 values
DLF_HD constexpr int tiles_q_buffers(int dp) { return dp <= 64 ? 3 : 1; }
DLF_HD constexpr int tiles_ring(int dp) { return dp <= 64 ? 7 : 4; }
DLF_HD constexpr int tiles_smem(int dp) { return 1024 + (tiles_q_buffers(dp) * 2 + tiles_ring(dp)) * (dp / 64) * kTileBlock; }
DLF_HD constexpr int tiles_slot(int size) { return 256 * (size + 2); }

__device__ __forceinline__ PlanWalk tiles_walk(const TilesParams& p) {
    return PlanWalk(PlanLengths{p.lengths, p.keys, p.batch, kTileKeys, p.status}, p.heads * p.q_pairs, p.ctas, 1);
}
// registers: 640 x 96 at launch; the softmax warps take 104, the others 64 (4 * 104 + 64 = 5 * 96)
constexpr int kTilesSoftmaxRegs = 104, kTilesOtherRegs = 64;

struct TilesItem {
    int head, row0, tile0, tiles;  // first tile of keys of the segment, and how many
    bool two;                      // the second tile of queries exists
};
__device__ __forceinline__ TilesItem tiles_item(const TilesParams& p, const PlanWalk& w) {
    TilesItem x;
    x.head = w.head / p.q_pairs;
    x.row0 = (w.head - x.head * p.q_pairs) * 256;
    x.two = x.row0 + 128 < p.queries;
    x.tile0 = w.unit0;
    x.tiles = w.count();
    return x;
}
// whether the tile has keys that do not count although they lie inside the tensors
__device__ __forceinline__ bool tiles_dirty(const TilesParams& p, int len, int tile) {
    return p.mask != nullptr || (len < p.keys && (tile + 1) * kTileKeys > len);
}
// keys of a tile, up to a multiple of 16: what the products are made over
__device__ __forceinline__ int tiles_depth(int len, int tile) { return (min(kTileKeys, len - tile * kTileKeys) + 15) & ~15; }

namespace ptx {
__device__ __forceinline__ float max_of(float a, float b, float c) {  // a NaN stays one
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
}  // namespace ptx

template <bool BF16, int DP>
__global__ void __launch_bounds__(kTilesThreads, 1)
    attention_tiles_kernel(const __grid_constant__ TilesParams p, const __grid_constant__ CUtensorMap tmQ,
                           const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                           const __grid_constant__ CUtensorMap tmY) {
    constexpr int DB = DP / 64, NQ = tiles_q_buffers(DP), R = tiles_ring(DP);
    constexpr uint32_t TILE = DB * kTileBlock;  // bytes of a tile of queries, keys or values
    constexpr int NS = DP <= 64 ? 2 : 1;        // regions of S
    static_assert(NS == 2 || NQ == 1, "the issuers rely on it");
    // The next segment's queries, first keys and first S come before this one's last values and product; not where the segments
    // share a Q buffer, which is free after that product only.
    constexpr bool AHEAD = NQ > 1;
    constexpr uint32_t kS = 0u, kP = NS * 128u, kO = kP + 128u;  // tensor-memory columns
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t q_full[NQ], q_empty[NQ], full_bar[R], empty_bar[R], fixed_bar[R], s_full[2], s_free[2], p_full[2], o_done[2], pair_bar[2][4];
    __shared__ float pair_value[2][2][2][128];  // parity of the exchange, tile, half, row
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t smem0 = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ring = smem0 + NQ * 2 * TILE;

    const bool zeroing = p.mask != nullptr || p.lengths != nullptr;  // there may be keys that do not count

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < NQ; ++i) {
            ptx::mbar_init(ptx::smem_u32(&q_full[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&q_empty[i]), 18u);  // the softmax warps and the issuers
        }
        for (int i = 0; i < R; ++i) {
            ptx::mbar_init(ptx::smem_u32(&full_bar[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&empty_bar[i]), zeroing ? 3u : 2u);  // the issuers and the warp that zeroes
            ptx::mbar_init(ptx::smem_u32(&fixed_bar[i]), 1u);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(ptx::smem_u32(&s_full[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&p_full[i]), 8u);
            ptx::mbar_init(ptx::smem_u32(&o_done[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&s_free[i]), 8u);
            for (int q = 0; q < 4; ++q) ptx::mbar_init(ptx::smem_u32(&pair_bar[i][q]), 2u);
        }
        ptx::fence_mbar_init();
    }
    if (warp == 16) {
        __syncwarp();
        ptx::tmem_alloc_then_dependents(ptx::smem_u32(&tmem_slot), 512u);
    }
    if (warp == 17 && lane == 0) {
        ptx::tma_prefetch_desc(&tmQ);
        ptx::tma_prefetch_desc(&tmK);
        ptx::tma_prefetch_desc(&tmV);
        ptx::tma_prefetch_desc(&tmY);
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
    volatile int* abort_p = &abort_flag;
    const long long limit = p.wait_limit;
    ptx::wait_for_dependencies();
    auto wait = [&](uint64_t& bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, ptx::mbar_wait_bounded(ptx::smem_u32(&bar), parity, abort_p, limit));
    };

    if (warp >= 16) {
        ptx::registers_down<kTilesOtherRegs>();
        PlanWalk walk = tiles_walk(p);
        if (walk.more() && walk.len <= 0) walk.next_with_keys();  // (rows without keys are the softmax warps' alone)
        if (warp == 17) {
            // -------------------------------------------------------- loads
            const bool leader = ptx::elect_one();
            uint32_t qb = 0, qph = 0, s = 0, ph = 0;
            auto load = [&](const CUtensorMap* map, int tile, int head, int batch) -> bool {
                if (!wait(empty_bar[s], ph ^ 1u)) return false;
                if (leader) {
                    const uint32_t bar = ptx::smem_u32(&full_bar[s]);
                    ptx::mbar_arrive_expect_tx(bar, TILE);
#pragma unroll
                    for (int db = 0; db < DB; ++db)
                        ptx::tma_load_4d(ring + s * TILE + db * kTileBlock, map, bar, db * 64, tile * kTileKeys, head, batch);
                }
                __syncwarp();
                if (++s == R) {
                    s = 0;
                    ph ^= 1u;
                }
                return true;
            };
            auto start = [&](const PlanWalk& at) -> bool {  // a segment's queries and first keys
                const TilesItem w = tiles_item(p, at);
                if (!wait(q_empty[qb], qph ^ 1u)) return false;
                if (leader) {
                    const uint32_t bar = ptx::smem_u32(&q_full[qb]);
                    ptx::mbar_arrive_expect_tx(bar, (w.two ? 2u : 1u) * TILE);
                    for (int t = 0; t < (w.two ? 2 : 1); ++t)
#pragma unroll
                        for (int db = 0; db < DB; ++db)
                            ptx::tma_load_4d(smem0 + (qb * 2 + t) * TILE + db * kTileBlock, &tmQ, bar, db * 64, w.row0 + t * 128, w.head,
                                             p.q_batched ? at.b : 0);
                }
                __syncwarp();
                if (++qb == NQ) {
                    qb = 0;
                    qph ^= 1u;
                }
                return load(&tmK, w.tile0, w.head / p.group, p.k_batched ? at.b : 0);
            };
            bool ok = !walk.more() || start(walk);
            while (ok && walk.more()) {
                const TilesItem w = tiles_item(p, walk);
                const int hk = w.head / p.group, kb = p.k_batched ? walk.b : 0, vb = p.v_batched ? walk.b : 0;
                for (int i = 0; ok && i + 1 < w.tiles; ++i) ok = load(&tmK, w.tile0 + i + 1, hk, kb) && load(&tmV, w.tile0 + i, hk, vb);
                walk.next_with_keys();
                const bool another = walk.more();
                if (AHEAD) ok = ok && (!another || start(walk));
                ok = ok && load(&tmV, w.tile0 + w.tiles - 1, hk, vb);
                if (!AHEAD) ok = ok && (!another || start(walk));
            }
        } else if (warp != 19) {
            // -------------------------------------------------------- products of tile t
            const int t = warp == 16 ? 0 : 1;
            const uint32_t idesc_o = ptx::make_idesc(BF16 ? 1u : 0u, 0u, 1u, 128u, DP);
            const uint64_t dq0 = ptx::make_smem_desc(smem0 + t * TILE, 16u, 1024u, 2u);
            const uint64_t dk0 = ptx::make_smem_desc(ring, 16u, 1024u, 2u);
            const uint64_t dv0 = ptx::make_smem_desc(ring, kTileBlock, 1024u, 2u);  // (MN-major: next 64 d's a block on)
            uint32_t qb = 0, qph = 0, s = 0, ph = 0, pph = 0, fixed_ph = 0;
            // How many S of tile 0 and 1 there have been (parity), and whose last one the next S waits for: with a region for each tile its
            // own; with one region tile 0 for tile 1's (its own where there is no tile 1), tile 1 for tile 0's of the same keys. The
            // phase waited for is never more than one ahead: in one region the tiles take turns, and a segment starts
            // (q_full, one buffer) when every S of the segment before it has been taken.
            uint32_t taken[2] = {0, 0};
            int last = -1;
            auto next_slot = [&]() {
                if (++s == R) {
                    s = 0;
                    ph ^= 1u;
                }
            };
            // S = Q K^T of a tile of keys, from slot s (tile 1 where there is none: the slot passes by, when it has been filled, or its phase
            // could not be told)
            auto scores = [&](const PlanWalk& at, bool two, int tile) -> bool {
                if (!wait(full_bar[s], ph)) return false;
                if (t == 1 && !two) {
                    taken[0] ^= 1u;
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&empty_bar[s]));
                    __syncwarp();
                    next_slot();
                    return true;
                }
                if (NS == 2) {
                    if (last >= 0 && !wait(s_free[t], taken[t] ^ 1u)) return false;
                    last = t;
                    taken[t] ^= 1u;
                } else {
                    if (t == 1) last = 0, taken[0] ^= 1u;  // (tile 0's S of the same keys)
                    if (last >= 0 && !wait(s_free[last], taken[last] ^ 1u)) return false;
                    if (t == 0) {
                        taken[0] ^= 1u;
                        if (two) taken[1] ^= 1u;
                        last = two ? 1 : 0;
                    }
                }
                ptx::tc_fence_after();
                if (ptx::elect_one()) {
                    const uint32_t idesc_s = ptx::make_idesc(BF16 ? 1u : 0u, 0u, 0u, 128u, static_cast<uint32_t>(tiles_depth(at.len, tile)));
                    const uint64_t dq = dq0 + ((qb * 2 * TILE) >> 4), dk = dk0 + ((s * TILE) >> 4);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        ptx::umma_f16(tmem + kS + (NS == 2 ? t * 128 : 0), dq + (k / 4) * (kTileBlock >> 4) + (k % 4) * 2,
                                      dk + (k / 4) * (kTileBlock >> 4) + (k % 4) * 2, idesc_s, k > 0 ? 1u : 0u);
                    ptx::umma_commit(ptx::smem_u32(&s_full[t]));
                    ptx::umma_commit(ptx::smem_u32(&empty_bar[s]));
                }
                __syncwarp();
                next_slot();
                return true;
            };
            auto start = [&](const PlanWalk& at) -> bool {  // a segment's first S
                const TilesItem w = tiles_item(p, at);
                if (!wait(q_full[qb], qph)) return false;
                ptx::tc_fence_after();
                return scores(at, w.two, w.tile0);
            };
            // O += P V of a tile of keys, from slot s
            auto sums = [&](int len, bool two, int tile, bool first, bool final) -> bool {
                if (tiles_dirty(p, len, tile)) {
                    if (!wait(fixed_bar[s], (fixed_ph >> s) & 1u)) return false;
                    fixed_ph ^= 1u << s;
                } else if (!wait(full_bar[s], ph)) {
                    return false;
                }
                if (t == 1 && !two) {
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&empty_bar[s]));
                    __syncwarp();
                    next_slot();
                    return true;
                }
                const uint64_t dv = dv0 + ((s * TILE) >> 4);
                const int steps = tiles_depth(len, tile) / 16;
                if (!wait(p_full[t], pph)) return false;
                pph ^= 1u;
                ptx::tc_fence_after();
                if (ptx::elect_one()) {
#pragma unroll
                    for (int k = 0; k < kTileKeys / 16; ++k)  // 16 keys a step
                        if (k < steps)
                            ptx::umma_f16_tmem(tmem + kO + t * DP, tmem + kP + t * 64 + k * 8, dv + k * (2048 >> 4), idesc_o, (!first || k > 0) ? 1u : 0u);
                    if (!final || !p.withhold) ptx::umma_commit(ptx::smem_u32(&o_done[t]));
                    ptx::umma_commit(ptx::smem_u32(&empty_bar[s]));
                }
                __syncwarp();
                next_slot();
                return true;
            };
            bool ok = !walk.more() || start(walk);
            while (ok && walk.more()) {
                const TilesItem w = tiles_item(p, walk);
                const int len = walk.len;
                for (int i = 0; ok && i + 1 < w.tiles; ++i)
                    ok = scores(walk, w.two, w.tile0 + i + 1) && sums(len, w.two, w.tile0 + i, i == 0, false);
                if (!ok) break;
                if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&q_empty[qb]));  // (every S of the segment has been issued)
                if (++qb == NQ) {
                    qb = 0;
                    qph ^= 1u;
                }
                walk.next_with_keys();
                const bool another = walk.more();
                if (AHEAD) ok = !another || start(walk);
                ok = ok && sums(len, w.two, w.tile0 + w.tiles - 1, w.tiles == 1, true);
                if (!AHEAD) ok = ok && (!another || start(walk));
            }
        } else {
            // -------------------------------------------------------- value rows of keys that do not count: zeros
            uint32_t s = 0, ph = 0;
            // every slot is waited for in its turn and given back, the ones that need nothing too: a phase can only be told from the one
            // before it
            auto pass = [&]() -> bool {
                if (!wait(full_bar[s], ph)) return false;
                if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&empty_bar[s]));
                __syncwarp();
                if (++s == R) {
                    s = 0;
                    ph ^= 1u;
                }
                return true;
            };
            auto clean = [&](int b, int len, int tile) -> bool {
                if (tiles_dirty(p, len, tile)) {
                    if (!wait(full_bar[s], ph)) return false;
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const int row = h * 32 + lane, key = tile * kTileKeys + row;
                        if (key >= len || (p.mask != nullptr && p.mask[b * p.mask_sb + key] == 0)) {
                            const uint32_t at = ring + s * TILE + row * 128;
#pragma unroll
                            for (int db = 0; db < DB; ++db)
#pragma unroll
                                for (int c = 0; c < 8; ++c)
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + db * kTileBlock + ((c ^ (lane & 7)) << 4)), "r"(0) : "memory");
                        }
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&fixed_bar[s]));
                }
                return pass();
            };
            bool ok = zeroing && walk.more() && pass();  // (the first keys)
            while (ok && walk.more()) {
                const TilesItem w = tiles_item(p, walk);
                const int b = walk.b, len = walk.len;
                for (int i = 0; ok && i + 1 < w.tiles; ++i) ok = pass() && clean(b, len, w.tile0 + i);
                walk.next_with_keys();
                const bool another = walk.more();
                if (AHEAD) ok = ok && (!another || pass());
                ok = ok && clean(b, len, w.tile0 + w.tiles - 1);
                if (!AHEAD) ok = ok && (!another || pass());
            }
        }
    } else {
        // ------------------------------------------------------------ softmax: tile t, keys 64 h .. of each tile of keys, rows 32 q ..
        ptx::registers_up<kTilesSoftmaxRegs>();
        PlanWalk walk = tiles_walk(p);
        const int t = warp >> 3, h = (warp >> 2) & 1, q = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
        const uint32_t tS = tmem + kS + (NS == 2 ? t * 128 : 0) + h * 64 + lanes;
        const uint32_t tP = tmem + kP + t * 64 + h * 32 + lanes;
        const uint32_t tO = tmem + kO + t * DP + h * (DP / 2) + lanes;  // this half's share of O when it is scaled or read
        uint32_t qb = 0, qph = 0, sph = 0, oph = 0, xph = 0;
        const float c = p.c;
        bool ok = true;
        // what the other half of the row has
        auto other = [&](float mine, float& theirs) -> bool {
            pair_value[xph][t][h][q * 32 + lane] = mine;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&pair_bar[t][q]));
            if (!wait(pair_bar[t][q], xph)) return false;
            theirs = pair_value[xph][t][h ^ 1][q * 32 + lane];
            xph ^= 1u;
            return true;
        };
        int storing = -1;  // Q buffer that a result is being stored from
        auto release = [&]() {
            if (storing < 0) return;
            if (lane == 0) {
                ptx::bulk_wait_group_read<0>();
                ptx::mbar_arrive(ptx::smem_u32(&q_empty[storing]));
            }
            __syncwarp();
            storing = -1;
        };
        // the products of the tile before are done
        bool done = true;
        auto before = [&]() -> bool {
            if (done) return true;
            done = true;
            if (!wait(o_done[t], oph)) return false;
            oph ^= 1u;
            ptx::tc_fence_after();
            return true;
        };
        // O and the sum to the result (m: +infinity where a score was that or NaN)
        auto finish = [&](const TilesItem& w, float m, float half) -> bool {
            float l = 0.0f;
            if (!other(half, l) || !before()) return false;
            l += half;
            if (m == INFINITY) l = __uint_as_float(0x7fc00000u);
            if (walk.whole()) {
                const bool none = m == -INFINITY;  // no key kept: zeros
                const float inv = 1.0f / l;
                // staged as the store's box: 32 rows of 64 values (lines of 128 bytes, 128-byte swizzle), or of 32 (64 and 64)
                const uint32_t block = smem0 + (qb * 2 + t) * TILE + h * (TILE / 2) + q * (32 * DP);
                const uint32_t line = block + lane * DP, sw = DP == 128 ? lane & 7u : (lane >> 1) & 3u;
#pragma unroll 1
                for (int d = 0; d < DP / 2; d += 16) {
                    uint32_t o[16];
                    ptx::tmem_ld_32x16(tO + d, o);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t u[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float a = __uint_as_float(o[8 * k + 2 * x]), b = __uint_as_float(o[8 * k + 2 * x + 1]);
                            u[x] = none ? 0u : pack_16<BF16>(a * inv, b * inv);
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(line + (((d / 8 + k) ^ sw) << 4)), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3])
                                     : "memory");
                    }
                }
                ptx::tc_fence_before();
                ptx::fence_proxy_async_smem();
                __syncwarp();
                const int row = w.row0 + t * 128 + q * 32;
                if (lane == 0 && row < p.queries && h * (DP / 2) < p.size) {
                    ptx::tma_store_4d(&tmY, block, h * (DP / 2), row, w.head, walk.b);
                    ptx::bulk_commit_group();
                }
                __syncwarp();
                storing = static_cast<int>(qb);  // (with several Q buffers the wait for the store comes a tile later)
                if (NQ == 1) release();
            } else {
                // O and the sum as they are, in 32 bits
                float* part = p.parts + static_cast<long long>(walk.slot()) * tiles_slot(p.size);
                const int r = t * 128 + q * 32 + lane;
                if (h == 0) {
                    part[256 * p.size + 2 * r] = m;
                    part[256 * p.size + 2 * r + 1] = l;
                }
#pragma unroll 1
                for (int d = 0; d < DP / 2; d += 16) {
                    uint32_t o[16];
                    ptx::tmem_ld_32x16(tO + d, o);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int x = 0; x < 16; x += 8) {
                        const int at = h * (DP / 2) + d + x;
                        if (at < p.size) {
                            *reinterpret_cast<uint4*>(part + r * p.size + at) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
                            *reinterpret_cast<uint4*>(part + r * p.size + at + 4) = make_uint4(o[x + 4], o[x + 5], o[x + 6], o[x + 7]);
                        }
                    }
                }
                ptx::tc_fence_before();
                if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&q_empty[qb]));
            }
            return true;
        };
        for (; ok && walk.more(); walk.next()) {
            const TilesItem w = tiles_item(p, walk);
            if (walk.len <= 0) {
                // a sequence without keys: its rows are zeros, and nobody else takes part
                const int row = w.row0 + t * 128 + q * 32 + lane;
                if (row < p.queries)
                    for (int d = h * (DP / 2); d < min(p.size, (h + 1) * (DP / 2)); d += 8)
                        *reinterpret_cast<uint4*>(p.y + (walk.b * p.y_sb + row * p.y_st + w.head * p.y_sh + d) * 2) = make_uint4(0u, 0u, 0u, 0u);
                __syncwarp();
                continue;
            }
            if (t == 0 || w.two) {
                float m = -INFINITY, l = 0.0f;
                bool bad = false;  // a score that is NaN or +infinity
                for (int i = 0; i < w.tiles; ++i) {
                    ok = wait(s_full[t], sph);
                    if (!ok) break;
                    sph ^= 1u;
                    ptx::tc_fence_after();
                    const int key0 = (w.tile0 + i) * kTileKeys + 64 * h, left = walk.len - key0;  // (left <= 0: none for this half)
                    uint32_t v[2][32];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (32 * j < left) ptx::tmem_ld_32x32(tS + 32 * j, v[j]);
                    ptx::tmem_ld_wait();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s_free[t]));
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (32 * j >= left || (p.mask == nullptr && 32 * (j + 1) <= left)) continue;
                        const int key = key0 + 32 * j + lane;
                        const bool in = key < walk.len && (p.mask == nullptr || p.mask[walk.b * p.mask_sb + key] != 0);
                        const unsigned bits = __ballot_sync(0xffffffffu, in);
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (!((bits >> x) & 1u)) v[j][x] = 0xff800000u;
                    }
                    float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (32 * j >= left) continue;
#pragma unroll
                        for (int x = 0; x < 32; x += 4) {
                            mx = ptx::max_of(mx, __uint_as_float(v[j][x]), __uint_as_float(v[j][x + 1]));
                            mx1 = ptx::max_of(mx1, __uint_as_float(v[j][x + 2]), __uint_as_float(v[j][x + 3]));
                        }
                    }
                    float theirs;
                    mx = ptx::max_of(mx, mx1, mx1);
                    ok = other(mx, theirs);
                    if (!ok) break;
                    mx = ptx::max_of(mx, theirs, theirs);
                    bad |= !(mx < INFINITY);
                    if (i == 0) {
                        m = mx;
                    } else {
                        const bool move = (mx - m) * c > 8.0f;
                        if (__any_sync(0xffffffffu, move)) {  // (the same in both halves)
                            ok = before();
                            if (!ok) break;
                            const float f = move ? ptx::exp2_approx((m - mx) * c) : 1.0f;
                            if (move) m = mx;
                            l *= f;
#pragma unroll 1
                            for (int d = 0; d < DP / 2; d += 16) {
                                uint32_t o[16];
                                ptx::tmem_ld_32x16(tO + d, o);
                                ptx::tmem_ld_wait();
#pragma unroll
                                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                                ptx::tmem_st_32x16(tO + d, o);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : m;
                    float factor = c, less = base * c;
                    if (__any_sync(0xffffffffu, fabsf(less) > 1024.0f)) {
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[j][x] = __float_as_uint((__uint_as_float(v[j][x]) - base) * c);
                        factor = 1.0f;
                        less = 0.0f;
                    }
                    const float add = decode_lift<BF16>() - less;
                    const uint64_t c2 = ptx::pair_of(factor, factor), add2 = ptx::pair_of(add, add);
                    uint64_t l2 = ptx::pair_of(0.0f, 0.0f), l3 = l2;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {  // 32 keys each
                        if (32 * j >= left) continue;
                        uint32_t o[16];
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            float a, b;
                            uint64_t s = ptx::fma_pair(ptx::pair_of(__uint_as_float(v[j][2 * x]), __uint_as_float(v[j][2 * x + 1])), c2, add2);
                            ptx::of_pair(s, a, b);
                            a = ptx::exp2_approx(a);
                            b = ptx::exp2_approx(b);
                            s = ptx::pair_of(a, b);
                            if (x & 1) l3 = ptx::add_pair(l3, s);
                            else l2 = ptx::add_pair(l2, s);
                            o[x] = pack_16<BF16>(a, b);
                        }
                        if (j == 0) ok = before();  // (they read the P that is replaced now)
                        if (!ok) break;
                        ptx::tmem_st_32x16(tP + 16 * j, o);
                    }
                    ok = ok && before();
                    if (!ok) break;
                    ptx::tmem_st_wait();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&p_full[t]));
                    done = false;
                    float la, lb;
                    ptx::of_pair(ptx::add_pair(l2, l3), la, lb);
                    l += la + lb;
                    release();
                }
                if (!ok) break;
                ok = finish(w, bad ? INFINITY : m, l);
                if (!ok) break;
            } else {
                // no second tile: the buffer is given back in this segment's turn
                release();
                ok = wait(q_full[qb], qph);
                if (!ok) break;
                if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&q_empty[qb]));
            }
            if (++qb == NQ) {
                qb = 0;
                qph ^= 1u;
            }
        }
        if (lane == 0) ptx::bulk_wait_group_read<0>();
    }
    __syncthreads();
    if (abort_flag) {
        // copies and UMMAs still in flight get time to land before shared and tensor memory are released
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        if (threadIdx.x == 0) atomicOr(p.status, 1);
    }
    if (warp == 16) {
        __syncwarp();
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512u);
    }
}

// Joins the parts of the (head, pair of query tiles) that the end of CTA blockIdx.x's range cuts, 16 rows a block; where a range's
// end cuts one that the end before it cuts too, that one has done it.
constexpr int kTilesJoinRows = 16;
template <bool BF16>
__global__ void __launch_bounds__(128) attention_tiles_join_kernel(const __grid_constant__ TilesParams p) {
    const PlanLengths lengths{p.lengths, p.keys, p.batch, kTileKeys, p.status};
    const int heads = p.heads * p.q_pairs;
    ptx::wait_for_dependencies();
    int before, all;
    plan_sums(lengths, 0, before, all);
    all *= heads;
    const int per = plan_per(all, p.ctas, 1);
    if ((blockIdx.x + 1ll) * per >= all) return;
    const int cut = (static_cast<int>(blockIdx.x) + 1) * per;
    const int b = plan_find(lengths, cut, heads, before);
    const int units = plan_units(plan_sequence(lengths, b), kTileKeys);
    const int item = (cut - before) / units;
    const int first = before + item * units, last = first + units - 1;
    if (first == cut || first < cut - per) return;  // not cut here; or cut earlier
    const int c0 = first / per, c1 = last / per;
    const int head = item / p.q_pairs, row0 = (item - head * p.q_pairs) * 256;
    const int chunks = p.size / 4;
    const long long slot_floats = tiles_slot(p.size);
    const float* first_part = p.parts + plan_slot(first, per) * slot_floats;
    for (int id = threadIdx.x; id < kTilesJoinRows * chunks; id += blockDim.x) {
        const int r = blockIdx.y * kTilesJoinRows + id / chunks, ch = id % chunks;
        if (row0 + r >= p.queries) continue;
        float mm = first_part[256 * p.size + 2 * r];
        for (int c = c0 + 1; c <= c1; ++c) mm = fmaxf(mm, p.parts[2ll * c * slot_floats + 256 * p.size + 2 * r]);
        float ll = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int c = c0; c <= c1; ++c) {
            const float* part = c == c0 ? first_part : p.parts + 2ll * c * slot_floats;
            const float f = mm == -INFINITY ? 0.0f : ptx::exp2_approx((part[256 * p.size + 2 * r] - mm) * p.c);
            const float4 x = *reinterpret_cast<const float4*>(part + r * p.size + ch * 4);
            ll += f * part[256 * p.size + 2 * r + 1];
            acc[0] += f * x.x;
            acc[1] += f * x.y;
            acc[2] += f * x.z;
            acc[3] += f * x.w;
        }
        const float inv = mm == -INFINITY ? 0.0f : 1.0f / ll;
        uint2 w;
        w.x = pack_16<BF16>(acc[0] * inv, acc[1] * inv);
        w.y = pack_16<BF16>(acc[2] * inv, acc[3] * inv);
        *reinterpret_cast<uint2*>(p.y + (b * p.y_sb + (row0 + r) * p.y_st + head * p.y_sh + ch * 4) * 2) = w;
    }
}

}  // namespace dlfb200
