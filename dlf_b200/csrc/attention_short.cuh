// Attention of many query rows over few keys: one tile of up to 128 keys (an image's or a decoder's positions over a short text).
//
//     S = Q K^T,  p = exp2(c (S - m)),  O = P V,  y = O / sum p      (c = scale * log2 e, m the largest score of the row)
//
// In fp16 p is taken times 2^15, the most that it holds (m is the largest score itself): its 11 bits then reach down to 2^-29 of the
// largest.
//
// All the keys are there at once, so there is no recurrence and nothing is cut. What is left is a chain for each tile of 128 queries -
// load, S, softmax, P V, store - that no unit fills, so what counts is how many tiles an SM has in flight, each at another place of its
// chain: small blocks of four softmax warps (a thread a query row) and one warp for loads and products, four to an SM with heads of 64.
//
// Tensor memory: S in 128 columns, and in its place, when a chunk of 32 scores has been read for the second time, P (16-bit pairs, each p
// rounded once as in attention_tiles.cuh, the A operand of P V; chunk j goes to columns 16 j .., all of them read by then). With heads of 64 O lies in columns 64 .. 127, which P
// leaves free; with heads of 128 behind S. The scores are read twice (maximum; exponentials): a whole row does not fit into the
// registers that four blocks leave.
//
// The difference is always taken first: the choice that attention_tiles.cuh makes by the size of c m costs more here than it saves (16 x
// 4096 queries over 128 keys, 8 heads of 64: 42.7 us with it, 41.8 without).
//
// 16 x 4096 queries over 77 keys, 8 heads: 34 us with heads of 64, 54 with heads of 128 (21 and 42 at the copy rate); attention_tiles.cuh,
// whose block has two tiles in flight that its barriers keep in step, takes 46 and 89.
//
// A block runs through consecutive tiles of queries, so the keys and values of a kv head are loaded once for all of a block's tiles of
// it; the next tile's queries are fetched beside this one's softmax, into the other of two buffers. The result is staged in the
// buffer that held the tile's queries and leaves by TMA stores, 32 rows a warp.
#pragma once
#include "attention_tiles.cuh"

namespace dlfb200 {

struct ShortParams {
    int batch, queries, keys, heads, group, size;
    const int* lengths;         // or null: `keys` each
    const unsigned char* mask;  // (batch, keys) or null
    long long mask_sb;
    int q_tiles, tiles, key_rows;  // tiles of 128 queries of a head, and of all; keys up to a multiple of 16
    int buffers;                   // of queries: 1 or 2
    int k_batched, v_batched, q_batched;
    float c;
    char* y;
    long long y_sb, y_st, y_sh;  // elements
    int* status;
    long long wait_limit;
    int withhold;  // test aid: the commit behind P V is left out
};

constexpr int kShortThreads = 160;
DLF_HD constexpr int short_ctas_per_sm(int dp) { return dp <= 64 ? 4 : 2; }
DLF_HD constexpr int short_columns(int dp) { return dp <= 64 ? 128 : 256; }
// (at least so much that no more blocks find room than tensor memory has columns for: one that waits for those would be a tile late)
DLF_HD constexpr int short_smem(int dp, int key_rows, int buffers) {
    const int need = 1024 + (dp / 64) * (buffers * kTileBlock + 2 * key_rows * 128), least = 228 * 1024 / (short_ctas_per_sm(dp) + 1);
    return need > least ? need : least;
}

template <bool BF16, int DP>
__global__ void __launch_bounds__(kShortThreads, short_ctas_per_sm(DP))
    attention_short_kernel(const __grid_constant__ ShortParams p, const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                           const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmY) {
    constexpr int DB = DP / 64;
    constexpr uint32_t TILE = DB * kTileBlock;
    constexpr uint32_t kO = DP <= 64 ? 64u : 128u;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full, v_full, s_full, p_full, o_full, o_read;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t smem0 = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t key_block = static_cast<uint32_t>(p.key_rows) * 128u;  // bytes of 64 values of every key
    const uint32_t skeys = smem0 + p.buffers * TILE, svalues = skeys + DB * key_block;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(ptx::smem_u32(&q_full[i]), 1u);
            ptx::mbar_init(ptx::smem_u32(&q_empty[i]), 4u);
        }
        ptx::mbar_init(ptx::smem_u32(&k_full), 1u);
        ptx::mbar_init(ptx::smem_u32(&v_full), 1u);
        ptx::mbar_init(ptx::smem_u32(&s_full), 1u);
        ptx::mbar_init(ptx::smem_u32(&p_full), 4u);
        ptx::mbar_init(ptx::smem_u32(&o_full), 1u);
        ptx::mbar_init(ptx::smem_u32(&o_read), 4u);
        ptx::fence_mbar_init();
    }
    if (warp == 4) {
        __syncwarp();
        ptx::tmem_alloc_then_dependents(ptx::smem_u32(&tmem_slot), short_columns(DP));
    }
    if (threadIdx.x == 0) {
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

    const PlanLengths lengths{p.lengths, p.keys, p.batch, kTileKeys, p.status};
    const int end = static_cast<int>((blockIdx.x + 1ll) * p.tiles / gridDim.x);
    struct Place {
        int tile, b, head, row0, len;
    };
    auto place = [&](int tile) -> Place {
        Place x;
        const int bh = tile / p.q_tiles;
        x.tile = tile;
        x.row0 = (tile - bh * p.q_tiles) * 128;
        x.b = bh / p.heads;
        x.head = bh - x.b * p.heads;
        x.len = tile < end ? plan_sequence(lengths, x.b) : 0;
        return x;
    };
    Place at = place(static_cast<int>(static_cast<long long>(blockIdx.x) * p.tiles / gridDim.x));
    // the n-th tile that has keys, its buffer and the parity of its phase there
    uint32_t n = 0;
    const bool two = p.buffers == 2;
    auto buffer = [&](uint32_t i) -> uint32_t { return two ? i & 1u : 0u; };
    auto phase = [&](uint32_t i) -> uint32_t { return two ? (i >> 1) & 1u : i & 1u; };
    int group = -1;        // (batch entry, kv head) that K and V are of
    uint32_t groups = 0;   // how many there have been

    if (warp == 4) {
        // ------------------------------------------------------------ loads and products
        const bool leader = ptx::elect_one();
        auto with_keys = [&](Place x) -> Place {
            while (x.tile < end && x.len <= 0) x = place(x.tile + 1);
            return x;
        };
        auto load_q = [&](const Place& x, uint32_t i) -> bool {
            if (!wait(q_empty[buffer(i)], phase(i) ^ 1u)) return false;
            if (leader) {
                const uint32_t bar = ptx::smem_u32(&q_full[buffer(i)]);
                ptx::mbar_arrive_expect_tx(bar, TILE);
#pragma unroll
                for (int db = 0; db < DB; ++db)
                    ptx::tma_load_4d(smem0 + buffer(i) * TILE + db * kTileBlock, &tmQ, bar, db * 64, x.row0, x.head, p.q_batched ? x.b : 0);
            }
            __syncwarp();
            return true;
        };
        auto load_keys = [&](const CUtensorMap* map, uint32_t to, uint64_t& full, int hk, int b) {
            if (leader) {
                const uint32_t bar = ptx::smem_u32(&full);
                ptx::mbar_arrive_expect_tx(bar, DB * key_block);
#pragma unroll
                for (int db = 0; db < DB; ++db) ptx::tma_load_4d(to + db * key_block, map, bar, db * 64, 0, hk, b);
            }
            __syncwarp();
        };
        const uint32_t idesc_o = ptx::make_idesc(BF16 ? 1u : 0u, 0u, 1u, 128u, DP);
        const uint64_t dk = ptx::make_smem_desc(skeys, 16u, 1024u, 2u), dv = ptx::make_smem_desc(svalues, key_block, 1024u, 2u);
        at = with_keys(at);
        bool ok = at.tile >= end || load_q(at, 0);
        while (ok && at.tile < end) {
            const int hk = at.head / p.group, kv = at.b * (p.heads / p.group) + hk;
            const bool fresh = kv != group;
            // the tile before: its O has been read, so its products are done, and S may take its place, others K and V
            if (n > 0 && !wait(o_read, (n - 1) & 1u)) break;
            if (fresh) {
                group = kv;
                ++groups;
                load_keys(&tmK, skeys, k_full, hk, p.k_batched ? at.b : 0);
                load_keys(&tmV, svalues, v_full, hk, p.v_batched ? at.b : 0);
                if (!wait(k_full, (groups - 1) & 1u)) break;
            }
            if (!wait(q_full[buffer(n)], phase(n))) break;
            ptx::tc_fence_after();
            const int depth = (at.len + 15) & ~15;
            if (leader) {
                const uint32_t idesc_s = ptx::make_idesc(BF16 ? 1u : 0u, 0u, 0u, 128u, static_cast<uint32_t>(depth));
                const uint64_t dq = ptx::make_smem_desc(smem0 + buffer(n) * TILE, 16u, 1024u, 2u);
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
                    ptx::umma_f16(tmem, dq + (k / 4) * (kTileBlock >> 4) + (k % 4) * 2, dk + (k / 4) * (key_block >> 4) + (k % 4) * 2, idesc_s, k > 0 ? 1u : 0u);
                ptx::umma_commit(ptx::smem_u32(&s_full));
            }
            __syncwarp();
            const Place next = with_keys(place(at.tile + 1));
            if (two && next.tile < end && !load_q(next, n + 1)) break;
            if (fresh && !wait(v_full, (groups - 1) & 1u)) break;
            if (!wait(p_full, n & 1u)) break;
            ptx::tc_fence_after();
            if (leader) {
#pragma unroll
                for (int k = 0; k < kTileKeys / 16; ++k)
                    if (k * 16 < depth) ptx::umma_f16_tmem(tmem + kO, tmem + k * 8, dv + k * (2048 >> 4), idesc_o, k > 0 ? 1u : 0u);
                if (!p.withhold) ptx::umma_commit(ptx::smem_u32(&o_full));
            }
            __syncwarp();
            if (!two && next.tile < end && !load_q(next, n + 1)) break;
            at = next;
            ++n;
        }
    } else {
        // ------------------------------------------------------------ softmax: rows 32 warp ..
        const uint32_t mine = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        const float c = p.c;
        int storing = -1;  // buffer that a result is being stored from
        auto release = [&]() {
            if (storing < 0) return;
            if (lane == 0) {
                ptx::bulk_wait_group_read<0>();
                ptx::mbar_arrive(ptx::smem_u32(&q_empty[storing]));
            }
            __syncwarp();
            storing = -1;
        };
        for (; at.tile < end; at = place(at.tile + 1)) {
            const int row = at.row0 + warp * 32;
            if (at.len <= 0) {
                // no keys: zeros, and nobody else takes part
                if (row + lane < p.queries)
                    for (int d = 0; d < p.size; d += 8)
                        *reinterpret_cast<uint4*>(p.y + (at.b * p.y_sb + (row + lane) * p.y_st + at.head * p.y_sh + d) * 2) = make_uint4(0u, 0u, 0u, 0u);
                __syncwarp();
                continue;
            }
            const int kv = at.b * (p.heads / p.group) + at.head / p.group;
            const bool fresh = kv != group;
            if (fresh) {
                group = kv;
                ++groups;
            }
            unsigned kept[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = 32 * j + lane;
                kept[j] = __ballot_sync(0xffffffffu, key < at.len && (p.mask == nullptr || p.mask[at.b * p.mask_sb + key] != 0));
            }
            if (!wait(s_full, n & 1u)) break;
            ptx::tc_fence_after();
            release();  // (the buffer of the tile before: its result has long left)
            float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (32 * j >= at.len) continue;
                uint32_t v[32];
                ptx::tmem_ld_32x32(mine + 32 * j, v);
                ptx::tmem_ld_wait();
                if (kept[j] != 0xffffffffu) {
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if (!((kept[j] >> x) & 1u)) v[x] = 0xff800000u;
                }
#pragma unroll
                for (int x = 0; x < 32; x += 4) {
                    mx = ptx::max_of(mx, __uint_as_float(v[x]), __uint_as_float(v[x + 1]));
                    mx1 = ptx::max_of(mx1, __uint_as_float(v[x + 2]), __uint_as_float(v[x + 3]));
                }
            }
            mx = ptx::max_of(mx, mx1, mx1);
            const float base = mx == -INFINITY ? 0.0f : mx;
            constexpr float kLift = BF16 ? 0.0f : 15.0f;
            const uint64_t c2 = ptx::pair_of(c, c), base2 = ptx::pair_of(-base, -base), lift2 = ptx::pair_of(kLift, kLift);
            uint64_t l2 = ptx::pair_of(0.0f, 0.0f), l3 = l2;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (32 * j >= at.len) continue;
                uint32_t v[32], o[16];
                ptx::tmem_ld_32x32(mine + 32 * j, v);
                ptx::tmem_ld_wait();
                if (kept[j] != 0xffffffffu) {
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if (!((kept[j] >> x) & 1u)) v[x] = 0xff800000u;
                }
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    float a, b;
                    uint64_t s = ptx::fma_pair(ptx::add_pair(ptx::pair_of(__uint_as_float(v[2 * x]), __uint_as_float(v[2 * x + 1])), base2), c2, lift2);
                    ptx::of_pair(s, a, b);
                    a = ptx::exp2_approx(a);
                    b = ptx::exp2_approx(b);
                    s = ptx::pair_of(a, b);
                    if (x & 1) l3 = ptx::add_pair(l3, s);
                    else l2 = ptx::add_pair(l2, s);
                    o[x] = pack_16<BF16>(a, b);
                }
                ptx::tmem_st_32x16(mine + 16 * j, o);
            }
            // the values of keys that do not count: zeros (0 * NaN would be NaN), a row a thread, once for all tiles that read them
            if (fresh && (p.mask != nullptr || at.len < p.keys)) {
                if (!wait(v_full, (groups - 1) & 1u)) break;
                const int key = warp * 32 + lane;
                const unsigned own = warp < 2 ? (warp == 0 ? kept[0] : kept[1]) : (warp == 2 ? kept[2] : kept[3]);
                if (key < p.key_rows && !((own >> lane) & 1u)) {
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int x = 0; x < 8; ++x)  // (starting at another piece in every line: no bank conflicts)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(svalues + db * key_block + key * 128 + ((x ^ (lane & 7)) << 4)), "r"(0) : "memory");
                }
                ptx::fence_proxy_async_smem();
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&p_full));
            float l, lb;
            ptx::of_pair(ptx::add_pair(l2, l3), l, lb);
            l += lb;
            if (!(mx < INFINITY)) l = __uint_as_float(0x7fc00000u);  // a score that is NaN or +infinity
            const bool none = mx == -INFINITY;                       // no key kept: zeros
            const float inv = 1.0f / l;
            if (!wait(o_full, n & 1u)) break;
            ptx::tc_fence_after();
            // staged as the store's boxes: 32 rows of 64 values (lines of 128 bytes, 128-byte swizzle)
            const uint32_t block = smem0 + buffer(n) * TILE + warp * 4096, line = block + lane * 128;
#pragma unroll
            for (int d = 0; d < DP; d += 32) {
                uint32_t o[32];
                ptx::tmem_ld_32x32(mine + kO + d, o);
                ptx::tmem_ld_wait();
                if (d + 32 == DP) {
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&o_read));
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t u[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        u[x] = none ? 0u : pack_16<BF16>(__uint_as_float(o[8 * k + 2 * x]) * inv, __uint_as_float(o[8 * k + 2 * x + 1]) * inv);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(line + (d / 64) * kTileBlock + ((((d & 63) / 8 + k) ^ (lane & 7)) << 4)), "r"(u[0]),
                                 "r"(u[1]), "r"(u[2]), "r"(u[3])
                                 : "memory");
                }
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row < p.queries) {
#pragma unroll
                for (int db = 0; db < DB; ++db) ptx::tma_store_4d(&tmY, block + db * kTileBlock, db * 64, row, at.head, at.b);
                ptx::bulk_commit_group();
            }
            __syncwarp();
            storing = static_cast<int>(buffer(n));
            if (!two) release();
            ++n;
        }
        if (lane == 0) ptx::bulk_wait_group_read<0>();
    }
    __syncthreads();
    if (abort_flag) {
        // copies and UMMAs still in flight get time to land before shared and tensor memory are released
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        if (threadIdx.x == 0) atomicOr(p.status, 1);
    }
    if (warp == 4) {
        __syncwarp();
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, short_columns(DP));
    }
}

}  // namespace dlfb200
