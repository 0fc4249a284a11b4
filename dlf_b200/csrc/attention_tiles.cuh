// Attention of many query rows: two tiles of 128 queries per CTA against tiles of 128 keys, on the tensor cores.
//
//     S = Q K^T,  p = exp2(c S - c m),  O = sum over key tiles of P V,  y = O / sum p      (c = scale * log2 e)
//
// m is a reference near the running maximum of a row: it is moved (and O and the sum scaled) only when the maximum has grown by
// more than 2^8 since, which exp2's range allows and which makes the pass over O rare.
//
// Tensor memory (512 columns): S of the two tiles (128 columns each), O of the two tiles (DP columns each). P replaces S as
// 16-bit pairs (64 columns) and is the A operand of P V from there, so the scores never touch shared memory. P is rounded to
// the 16-bit type (the tensor core takes both operands of one type); O and the sums are 32-bit.
//
// Roles: warps 0-3 and 4-7 the softmax of tile 0 and 1 (a thread per query row), 8 UMMA issuer and TMEM owner, 9 TMA loads, 10 and
// 11 zero the value rows of keys that do not count (0 * NaN would be NaN). The issuer alternates the tiles -
// P0 V, next S0, P1 V, next S1 - so that one tile's softmax runs beside the other's products. K and V tiles go through one
// ring in the order of their use: K0, K1, V0, K2, V1, ... A CTA walks through its items (batch, head, pair of query tiles); the
// next item's loads and first products run beside this one's last. The result is staged in the item's own Q buffer and leaves
// by TMA stores, 32 rows a warp.
#pragma once
#include <cuda.h>

#include "attention_decode.cuh"
#include "attention_plan.h"
#include "dependents.cuh"
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
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void of_pair(uint64_t d, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(d)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
}  // namespace ptx

struct TilesParams {
    int batch, queries, keys, heads, kv_heads, group, size;
    const int* lengths;         // or null: `keys` each
    const unsigned char* mask;  // (batch, keys) or null
    long long mask_sb;
    int q_pairs, items;
    int k_batched, v_batched, q_batched;  // 0: the operand is shared by the batch
    float c;
    int* status;
    long long wait_limit;
    int withhold;  // test aid: the commit that ends the item is left out
};

constexpr int kTilesThreads = 384;
constexpr int kTileKeys = 128;
constexpr int kTileBlock = 128 * 128;  // bytes of 128 rows x 64 values
DLF_HD constexpr int tiles_q_buffers(int dp) { return dp <= 64 ? 2 : 1; }
DLF_HD constexpr int tiles_ring(int dp) { return dp <= 64 ? 8 : 5; }
DLF_HD constexpr int tiles_smem(int dp) { return 1024 + (tiles_q_buffers(dp) * 2 + tiles_ring(dp)) * (dp / 64) * kTileBlock; }
// registers: 384 x 168 at launch; the softmax warps take 208, the others 88 (2 * 208 + 88 = 3 * 168)
constexpr int kTilesSoftmaxRegs = 208, kTilesOtherRegs = 88;

struct TilesItem {
    int b, head, row0, len, tiles;  // tiles of keys
    bool two;                       // the second tile of queries exists
};
__device__ __forceinline__ TilesItem tiles_item(const TilesParams& p, int item) {
    TilesItem w;
    const int qp = item % p.q_pairs, r = item / p.q_pairs;
    w.b = r / p.heads;
    w.head = r - w.b * p.heads;
    w.row0 = qp * 256;
    w.len = p.keys;
    if (p.lengths != nullptr) {
        bool bad = false;
        w.len = plan_length(p.lengths[w.b], p.keys, &bad);
        if (bad && (threadIdx.x & 31) == 0) atomicOr(p.status, DEV_STATUS_BAD_PAGE);
    }
    w.tiles = (w.len + kTileKeys - 1) / kTileKeys;
    w.two = w.row0 + 128 < p.queries;
    return w;
}
// whether the tile has keys that do not count although they lie inside the tensors
__device__ __forceinline__ bool tiles_dirty(const TilesParams& p, const TilesItem& w, int i) {
    return p.mask != nullptr || (w.len < p.keys && (i + 1) * kTileKeys > w.len);
}

template <bool BF16, int DP>
__global__ void __launch_bounds__(kTilesThreads, 1)
    attention_tiles_kernel(const __grid_constant__ TilesParams p, const __grid_constant__ CUtensorMap tmQ,
                           const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                           const __grid_constant__ CUtensorMap tmY) {
    constexpr int DB = DP / 64, NQ = tiles_q_buffers(DP), R = tiles_ring(DP);
    constexpr uint32_t TILE = DB * kTileBlock;  // bytes of a tile of queries, keys or values
    constexpr uint32_t kS = 0u, kO = 256u;      // tensor-memory columns
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t q_full[NQ], q_empty[NQ], full_bar[R], empty_bar[R], fixed_bar[R], s_full[2], p_full[2], o_full[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t smem0 = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ring = smem0 + NQ * 2 * TILE;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < NQ; ++i) {
            ptx::mbar_init(ptx::smem_u32(&q_full[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&q_empty[i]), 9u);  // eight softmax warps and the issuer
        }
        for (int i = 0; i < R; ++i) {
            ptx::mbar_init(ptx::smem_u32(&full_bar[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&empty_bar[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&fixed_bar[i]), 2u);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(ptx::smem_u32(&s_full[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&p_full[i]), 4u);
            ptx::mbar_init(ptx::smem_u32(&o_full[i]), 1u);
        }
        ptx::fence_mbar_init();
    }
    if (warp == 8) {
        __syncwarp();
        ptx::tmem_alloc_then_dependents(ptx::smem_u32(&tmem_slot), 512u);
    }
    if (warp == 9 && lane == 0) {
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

    if (warp >= 8) {
        ptx::registers_down<kTilesOtherRegs>();
        if (warp == 9) {
            // -------------------------------------------------------- loads
            const bool leader = ptx::elect_one();
            uint32_t qb = 0, qph = 0, s = 0, ph = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < p.items; item += gridDim.x) {
                const TilesItem w = tiles_item(p, item);
                const int hk = w.head / p.group;
                auto load = [&](const CUtensorMap* map, int tile, int batch) -> bool {
                    if (!wait(empty_bar[s], ph ^ 1u)) return false;
                    if (leader) {
                        const uint32_t bar = ptx::smem_u32(&full_bar[s]);
                        ptx::mbar_arrive_expect_tx(bar, TILE);
#pragma unroll
                        for (int db = 0; db < DB; ++db)
                            ptx::tma_load_4d(ring + s * TILE + db * kTileBlock, map, bar, db * 64, tile * kTileKeys, hk, batch);
                    }
                    __syncwarp();
                    if (++s == R) {
                        s = 0;
                        ph ^= 1u;
                    }
                    return true;
                };
                if (!wait(q_empty[qb], qph ^ 1u)) break;
                if (leader) {
                    const uint32_t bar = ptx::smem_u32(&q_full[qb]);
                    ptx::mbar_arrive_expect_tx(bar, (w.two ? 2u : 1u) * TILE);
                    for (int t = 0; t < (w.two ? 2 : 1); ++t)
#pragma unroll
                        for (int db = 0; db < DB; ++db)
                            ptx::tma_load_4d(smem0 + (qb * 2 + t) * TILE + db * kTileBlock, &tmQ, bar, db * 64, w.row0 + t * 128, w.head,
                                             p.q_batched ? w.b : 0);
                }
                __syncwarp();
                if (++qb == NQ) {
                    qb = 0;
                    qph ^= 1u;
                }
                const int kb = p.k_batched ? w.b : 0, vb = p.v_batched ? w.b : 0;
                if (w.tiles > 0) ok = load(&tmK, 0, kb);
                for (int i = 0; ok && i < w.tiles; ++i) ok = (i + 1 == w.tiles || load(&tmK, i + 1, kb)) && load(&tmV, i, vb);
            }
        } else if (warp == 8) {
            // -------------------------------------------------------- products
            const uint32_t idesc_s = ptx::make_idesc(BF16 ? 1u : 0u, 0u, 0u, 128u, kTileKeys);
            const uint32_t idesc_o = ptx::make_idesc(BF16 ? 1u : 0u, 0u, 1u, 128u, DP);
            const uint64_t dq0 = ptx::make_smem_desc(smem0, 16u, 1024u, 2u);
            const uint64_t dk0 = ptx::make_smem_desc(ring, 16u, 1024u, 2u);
            const uint64_t dv0 = ptx::make_smem_desc(ring, kTileBlock, 1024u, 2u);  // (MN-major: next 64 d's a block on)
            uint32_t qb = 0, qph = 0, s = 0, ph = 0, pph[2] = {0, 0}, fixed_ph = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < p.items; item += gridDim.x) {
                const TilesItem w = tiles_item(p, item);
                const int nt = w.two ? 2 : 1;
                if (!wait(q_full[qb], qph)) break;
                ptx::tc_fence_after();
                auto scores = [&](int t, uint32_t slot) {  // S_t = Q_t K^T (by one thread)
                    const uint64_t dq = dq0 + (((qb * 2 + t) * TILE) >> 4), dk = dk0 + ((slot * TILE) >> 4);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        ptx::umma_f16(tmem + kS + t * 128, dq + (k / 4) * (kTileBlock >> 4) + (k % 4) * 2,
                                      dk + (k / 4) * (kTileBlock >> 4) + (k % 4) * 2, idesc_s, k > 0 ? 1u : 0u);
                    ptx::umma_commit(ptx::smem_u32(&s_full[t]));
                };
                auto next_slot = [&]() {
                    if (++s == R) {
                        s = 0;
                        ph ^= 1u;
                    }
                };
                if (w.tiles > 0) {
                    if (!wait(full_bar[s], ph)) break;
                    ptx::tc_fence_after();
                    if (ptx::elect_one()) {
                        for (int t = 0; t < nt; ++t) scores(t, s);
                        ptx::umma_commit(ptx::smem_u32(&empty_bar[s]));
                    }
                    __syncwarp();
                    next_slot();
                }
                for (int i = 0; i < w.tiles; ++i) {
                    const bool more = i + 1 < w.tiles;
                    const uint32_t ks = s;
                    if (more) {
                        ok = wait(full_bar[s], ph);
                        if (!ok) break;
                        next_slot();
                    }
                    const uint32_t vs = s;
                    if (tiles_dirty(p, w, i)) {
                        ok = wait(fixed_bar[s], (fixed_ph >> s) & 1u);
                        fixed_ph ^= 1u << s;
                    } else {
                        ok = wait(full_bar[s], ph);
                    }
                    if (!ok) break;
                    next_slot();
                    for (int t = 0; t < nt; ++t) {
                        ok = wait(p_full[t], pph[t]);
                        if (!ok) break;
                        pph[t] ^= 1u;
                        ptx::tc_fence_after();
                        if (ptx::elect_one()) {
                            const uint64_t dv = dv0 + ((vs * TILE) >> 4);
#pragma unroll
                            for (int k = 0; k < kTileKeys / 16; ++k)
                                ptx::umma_f16_tmem(tmem + kO + t * DP, tmem + kS + t * 128 + k * 8, dv + k * (2048 >> 4), idesc_o,
                                                   (i > 0 || k > 0) ? 1u : 0u);
                            if (more) scores(t, ks);
                            else if (!p.withhold) ptx::umma_commit(ptx::smem_u32(&o_full[t]));
                            if (t == nt - 1) {
                                if (more) ptx::umma_commit(ptx::smem_u32(&empty_bar[ks]));
                                ptx::umma_commit(ptx::smem_u32(&empty_bar[vs]));
                            }
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                }
                if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&q_empty[qb]));
                if (++qb == NQ) {
                    qb = 0;
                    qph ^= 1u;
                }
            }
        } else {
            // -------------------------------------------------------- value rows of keys that do not count: zeros
            const int half = warp - 10;
            uint32_t s = 0, ph = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < p.items; item += gridDim.x) {
                const TilesItem w = tiles_item(p, item);
                if (w.tiles == 0) continue;
                // every slot is waited for in its turn, the ones that need nothing too: a phase is told from the one before it only
                auto next = [&]() {
                    if (++s == R) {
                        s = 0;
                        ph ^= 1u;
                    }
                };
                auto pass = [&]() -> bool {
                    if (!wait(full_bar[s], ph)) return false;
                    next();
                    return true;
                };
                ok = pass();  // K0
                for (int i = 0; ok && i < w.tiles; ++i) {
                    if (i + 1 < w.tiles) ok = pass();
                    ok = ok && wait(full_bar[s], ph);
                    if (!ok) break;
                    if (tiles_dirty(p, w, i)) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int row = half * 64 + h * 32 + lane, key = i * kTileKeys + row;
                            if (key >= w.len || (p.mask != nullptr && p.mask[w.b * p.mask_sb + key] == 0)) {
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
                    next();
                }
            }
        }
    } else {
        // ------------------------------------------------------------ softmax
        ptx::registers_up<kTilesSoftmaxRegs>();
        const int t = warp >> 2, q = warp & 3;
        const uint32_t tS = tmem + kS + t * 128 + (static_cast<uint32_t>(q * 32) << 16);
        const uint32_t tO = tmem + kO + t * DP + (static_cast<uint32_t>(q * 32) << 16);
        uint32_t qb = 0, qph = 0, sph = 0, oph = 0;
        const float c = p.c;
        bool ok = true;
        for (int item = blockIdx.x; ok && item < p.items; item += gridDim.x) {
            const TilesItem w = tiles_item(p, item);
            if (t == 0 || w.two) {
                float m = -INFINITY, l = 0.0f;
                for (int i = 0; i < w.tiles; ++i) {
                    ok = wait(s_full[t], sph);
                    if (!ok) break;
                    sph ^= 1u;
                    ptx::tc_fence_after();
                    uint32_t v[4][32];
#pragma unroll
                    for (int j = 0; j < 4; ++j) ptx::tmem_ld_32x32(tS + 32 * j, v[j]);
                    ptx::tmem_ld_wait();
                    const int left = w.len - i * kTileKeys;
                    if (p.mask != nullptr || left < kTileKeys) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = i * kTileKeys + 32 * j + lane;
                            const bool in = key < w.len && (p.mask == nullptr || p.mask[w.b * p.mask_sb + key] != 0);
                            const unsigned bits = __ballot_sync(0xffffffffu, in);
#pragma unroll
                            for (int x = 0; x < 32; ++x)
                                if (!((bits >> x) & 1u)) v[j][x] = 0xff800000u;
                        }
                    }
                    float mx4[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mx4[j] = __uint_as_float(v[j][0]);
#pragma unroll
                        for (int x = 1; x < 32; ++x) mx4[j] = fmaxf(mx4[j], __uint_as_float(v[j][x]));
                    }
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                    if (i == 0) {
                        m = mx;
                    } else {
                        const bool move = (mx - m) * c > 8.0f;
                        if (__any_sync(0xffffffffu, move)) {
                            // (the products that O stands in are done: their commit is the one that S came with)
                            const float f = move ? ptx::exp2_approx((m - mx) * c) : 1.0f;
                            if (move) m = mx;
                            l *= f;
#pragma unroll 1
                            for (int d = 0; d < DP; d += 32) {
                                uint32_t o[32];
                                ptx::tmem_ld_32x32(tO + d, o);
                                ptx::tmem_ld_wait();
#pragma unroll
                                for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                                ptx::tmem_st_32x32(tO + d, o);
                            }
                        }
                    }
                    const float mc = m == -INFINITY ? 0.0f : m * c;
                    const uint64_t c2 = ptx::pair_of(c, c), mc2 = ptx::pair_of(-mc, -mc);
                    uint64_t l2 = ptx::pair_of(0.0f, 0.0f), l3 = l2;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t o[32];
#pragma unroll
                        for (int x = 0; x < 32; ++x) {
                            const int e = 2 * x;
                            float a = __uint_as_float(v[2 * j + e / 32][e % 32]), b = __uint_as_float(v[2 * j + e / 32][e % 32 + 1]);
                            ptx::of_pair(ptx::fma_pair(ptx::pair_of(a, b), c2, mc2), a, b);
                            a = ptx::exp2_approx(a);
                            b = ptx::exp2_approx(b);
                            if (x & 1) l3 = ptx::add_pair(l3, ptx::pair_of(a, b));
                            else l2 = ptx::add_pair(l2, ptx::pair_of(a, b));
                            o[x] = pack_16<BF16>(a, b);
                        }
                        ptx::tmem_st_32x32(tS + 32 * j, o);
                    }
                    float la, lb;
                    ptx::of_pair(ptx::add_pair(l2, l3), la, lb);
                    l += la + lb;
                    ptx::tmem_st_wait();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&p_full[t]));
                }
                if (!ok) break;
                // ---------------------------------------------------- the item's rows
                if (w.tiles > 0) {
                    ok = wait(o_full[t], oph);
                    oph ^= 1u;
                } else {
                    ok = wait(q_full[qb], qph);  // (the staging below must not meet the load)
                }
                if (!ok) break;
                ptx::tc_fence_after();
                const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // no key kept: zeros; a NaN stays one
                const uint32_t line = smem0 + (qb * 2 + t) * TILE + (q * 32 + lane) * 128;
#pragma unroll 1
                for (int d = 0; d < DP; d += 32) {
                    uint32_t o[32];
                    if (w.tiles > 0) {
                        ptx::tmem_ld_32x32(tO + d, o);
                        ptx::tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = 0u;
                    }
                    const bool none = l == 0.0f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t u[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float a = __uint_as_float(o[8 * k + 2 * x]), b = __uint_as_float(o[8 * k + 2 * x + 1]);
                            u[x] = none ? 0u : pack_16<BF16>(a * inv, b * inv);
                        }
                        const uint32_t ch = static_cast<uint32_t>((d % 64) / 8 + k);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(line + (d / 64) * kTileBlock + ((ch ^ (lane & 7u)) << 4)), "r"(u[0]),
                                     "r"(u[1]), "r"(u[2]), "r"(u[3])
                                     : "memory");
                    }
                }
                ptx::tc_fence_before();
                ptx::fence_proxy_async_smem();
                __syncwarp();
                const int row = w.row0 + t * 128 + q * 32;
                if (lane == 0 && row < p.queries) {
#pragma unroll
                    for (int db = 0; db < DB; ++db)
                        if (db * 64 < p.size)
                            ptx::tma_store_4d(&tmY, smem0 + (qb * 2 + t) * TILE + db * kTileBlock + q * 4096, db * 64, row, w.head, w.b);
                    ptx::bulk_commit_group();
                    ptx::bulk_wait_group_read<0>();
                }
                __syncwarp();
            } else {
                ok = wait(q_full[qb], qph);  // (its arrival below belongs to this item's use of the buffer)
                if (!ok) break;
            }
            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&q_empty[qb]));
            if (++qb == NQ) {
                qb = 0;
                qph ^= 1u;
            }
        }
    }
    __syncthreads();
    if (abort_flag) {
        // copies and UMMAs still in flight get time to land before shared and tensor memory are released
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        if (threadIdx.x == 0) atomicOr(p.status, 1);
    }
    if (warp == 8) {
        __syncwarp();
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512u);
    }
}

}  // namespace dlfb200
