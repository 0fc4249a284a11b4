// Attention of few query rows over many keys: one new token (or a few) of each sequence over a paged cache or over an
// encoder's states.
//
//     y_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp2(c (q_r.k_j - m_r)),  c = scale * log2(e),  m_r the largest so far
//
// The difference is taken before it is multiplied: of c s - c m in one fused step (c m rounded) the rounding of c m would be
// left, which for scores beyond 2^30 / c is more than exp2's range. Parts of a sequence are joined by the same rule, so m itself is
// what they leave beside their sums.
//
// HBM-bound: the keys and values of a kv head are read once for up to 16 query rows (the query heads that share it), so
// what counts is how many bytes are in flight and how few instructions a key costs. A block has four warps; of a unit of 64
// keys each takes 16 and runs the recurrence by itself (running maximum and sum, 32-bit accumulators), with its own ring of
// cp.async copies; the warps meet at the end of a segment (attention_plan.h).
//
// Products are mma.m16n8k16 with the keys (or the head's d's) as the 16 rows and the queries as the 8 columns, so up to
// eight query rows cost one set of instructions, up to 16 two (NB):
//   S^T = K Q^T: with g = lane / 4, t = lane % 4, lane (g, t) copies the 16-byte pieces t + 4 j of keys g and 8 + g and reads back
//      the same pieces: their four words are its fragments of two k-steps, if q's are taken in the same order of d's (a sum
//      over d has no order). No exchange, no bank conflicts.
//   O^T += V^T P^T: V's fragments by ldmatrix.trans (lines swizzled by the key), P^T by movmatrix from S^T's accumulators.
// The maximum of a row is moved (and O scaled) only when a score exceeds it by more than 2^8; until then a step needs no exchange
// between lanes. p is rounded to 16 bits for the second product in two parts (its rounding and the rest: 22 bits of fp16, 16 of bf16).
// fp16 ends at 2^-24, so there p is taken times 2^7 - up to 2^15 with the growth above - and what is lost lies below 2^-32 of the
// row's largest instead of 2^-25 (a key that outweighs the others by e^17.5 each made those of its warp nothing). The factor is the same
// everywhere and leaves with the division by the sum.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_plan.h"
#include "ptx.cuh"

namespace dlfb200 {

struct DecodeParams {
    const char* q;  // (batch, tokens, heads, size)
    const char* k;
    const char* v;
    char* y;
    long long q_sb, q_st, q_sh, y_sb, y_st, y_sh;  // elements
    long long k_sb, k_st, k_sh, v_sb, v_st, v_sh;  // paged: _sb a page's stride, _st a token's within its page
    const int* lengths;                            // or null: `keys` each
    const unsigned char* mask;                     // (batch, keys) or null
    long long mask_sb;
    const int* table;                              // page table (batch, table_width) or null
    long long table_sb;
    int page_size, num_pages;
    int batch, tokens, kv_heads, group, size, keys;
    int row_blocks, block_rows;                    // blocks of 8 or 16 rows (row = token * group + head of the group)
    int ctas, least;
    float c;                                       // scale * log2(e)
    float* parts;                                  // slots of 16 x (size + 2) floats: sums, then maximum and sum of p per row
    int4* cuts;                                    // for each CTA: what its end cuts (decode_cut)
    int* status;
};

// where a sequence's keys lie: one after the other; in pages of a multiple of 16 tokens (a step's 16 keys lie in one page); in
// pages of any size, or under a mask (every key by itself)
enum : int { KEYS_PLAIN = 0, KEYS_PAGES_16 = 1, KEYS_ANY = 2 };

constexpr float kLowest = -3.402823466e38f;  // below every score that counts; finite, so that differences from it are none of inf - inf

constexpr int kDecodeUnit = 64;  // keys
constexpr int kDecodeThreads = 128;
constexpr int kDecodeWarps = kDecodeThreads / 32;
// Stages of a warp's ring and blocks of an SM: nb = 1 or 2 sets of eight query rows. More blocks with shorter rings carry short
// segments better (32 sequences of up to 1500 keys, 16 heads of 64: 4 blocks of 3 stages 27.8 us, 3 of 4 29.2, 2 of 6 33.3), and cost long
// ones nothing (64 of up to 8192 keys, 8 heads of 128: 3 blocks of 2 stages 182.5 us, 2 of 3 184.4).
DLF_HD constexpr int decode_ctas_per_sm(int dp, int nb) { return dp <= 64 ? (nb == 1 ? 4 : 3) : (nb == 1 ? 3 : 2); }
DLF_HD constexpr int decode_stages(int dp, int nb) { return dp <= 64 ? (nb == 1 ? 3 : 4) : (nb == 1 ? 2 : 3); }
DLF_HD constexpr int decode_stage_bytes(int dp) { return 16 * dp * 2 * 2; }  // a warp's 16 keys and values
DLF_HD constexpr int decode_smem(int dp, int nb) { return kDecodeWarps * decode_stages(dp, nb) * decode_stage_bytes(dp); }
DLF_HD constexpr int decode_slot(int size) { return 16 * (size + 2); }
// A (sequence, head) that starts in a CTA's range and does not end there: sequence, head, slot of its first part, last CTA that
// has a part of it (their slots are 2 c). No sequence: -1.
__device__ __forceinline__ int4 decode_cut(const PlanWalk& w) {
    return make_int4(w.b, w.head, w.slot(), (w.u + w.units - 1) / w.per);
}

template <bool BF16>
DLF_HD constexpr float decode_lift() { return BF16 ? 0.0f : 7.0f; }  // p is taken times 2 to this

namespace ptx {
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool valid) {  // not valid: zeros, nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint4 lds_128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
}  // namespace ptx

template <bool BF16>
__device__ __forceinline__ uint32_t pack_16(float lo, float hi) {
    if constexpr (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack_16(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ PlanLengths decode_lengths(const DecodeParams& p) { return PlanLengths{p.lengths, p.keys, p.batch, kDecodeUnit, p.status}; }

template <bool BF16, int DP, int KEYS, int NB, bool FULL>  // FULL: the head has all DP values
__global__ void __launch_bounds__(kDecodeThreads, decode_ctas_per_sm(DP, NB)) attention_decode_kernel(const __grid_constant__ DecodeParams p) {
    constexpr int STAGES = decode_stages(DP, NB);
    constexpr int PK = DP / 32;  // pieces of a key per lane: t + 4 j, j < PK
    constexpr int PV = DP / 64;  // pieces of a value per lane: lane % 8 + 8 j
    constexpr int STAGE = decode_stage_bytes(DP), VOFF = STAGE / 2, LINE = DP * 2;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = ptx::smem_u32(smem_raw) + warp * STAGES * STAGE;
    // V: copied as piece lane % 8 + 8 j of keys lane / 8 + 4 i, to line `key`, piece ^ (key % 8)
    const int vkey = lane >> 3, vch = lane & 7;
    // read by ldmatrix: lane's line is key (lane & 7) + 8 for lanes 16.., piece + 1 for lanes 8-15 and 24-31
    const int mkey = (lane & 7) + ((lane >> 4) << 3), mch = (lane >> 3) & 1;
    const uint32_t vread = VOFF + mkey * LINE;

    ptx::wait_for_dependencies();
    ptx::launch_dependents();  // (behind the wait: what runs before this kernel is done when the joining one starts)

    PlanWalk walk(decode_lengths(p), p.kv_heads * p.row_blocks, p.ctas, p.least);
    const int chunks = p.size / 8;
    const float c = p.c;
    bool bad_page = false;
    int4 cut = make_int4(-1, 0, 0, 0);

    for (; walk.more(); walk.next()) {
        const int n_units = walk.count(), b = walk.b, len = walk.len, unit0 = walk.unit0;
        const bool whole = walk.whole();
        if (unit0 == 0 && !whole) cut = decode_cut(walk);  // (the last segment)
        const int hk = walk.head / p.row_blocks, row0 = (walk.head - hk * p.row_blocks) * p.block_rows;
        const int rows = min(8 * NB, p.tokens * p.group - row0);
        // ---------------------------------------------------------------- copies
        // step i of this warp: keys first_key + 64 i .. + 15
        const int first_key = unit0 * kDecodeUnit + warp * 16;
        const long long kst = p.k_st * 2, vst = p.v_st * 2;  // bytes between tokens
        const char* kbase = p.k + (p.table != nullptr ? 0 : b * p.k_sb * 2) + hk * p.k_sh * 2 + t * 16;
        const char* vbase = p.v + (p.table != nullptr ? 0 : b * p.v_sb * 2) + hk * p.v_sh * 2 + vch * 16;
        // what a step needs to know before it can be fetched: KEYS_PAGES_16 its page, KEYS_ANY lane l < 16 the place of key l (-1: not
        // kept). Asked for a step ahead of the fetch.
        auto ask = [&](int i) -> long long {
            const int pos = first_key + i * kDecodeUnit + (KEYS == KEYS_ANY ? (lane & 15) : 0);
            if (KEYS == KEYS_PLAIN || i >= n_units || pos >= len) return -1;
            if (KEYS == KEYS_PAGES_16 || p.table != nullptr) {
                const int pg = pos / p.page_size;
                const long long at = plan_place(p.table[b * p.table_sb + pg], pos - pg * p.page_size, p.num_pages);
                if (at < 0) bad_page = true;
                return at;
            }
            return p.mask[b * p.mask_sb + pos] == 0 ? -1 : pos;
        };
        // step i to a stage; returns which of its 16 keys count
        auto fetch = [&](int stage, int i, long long at) -> unsigned {
            const uint32_t kdst = ring + stage * STAGE + lane * 16;
            const uint32_t vdst = ring + stage * STAGE + VOFF + vkey * LINE;
            const int left = len - (first_key + i * kDecodeUnit);
            if constexpr (KEYS != KEYS_ANY) {
                const char* kp = kbase + g * kst;
                const char* vp = vbase + vkey * vst;
                if constexpr (KEYS == KEYS_PAGES_16) {
                    kp += ((at >> 32) * p.k_sb + static_cast<int>(at) * p.k_st) * 2;
                    vp += ((at >> 32) * p.v_sb + static_cast<int>(at) * p.v_st) * 2;
                } else {
                    kp += (first_key + static_cast<long long>(i) * kDecodeUnit) * kst;
                    vp += (first_key + static_cast<long long>(i) * kDecodeUnit) * vst;
                }
                if (FULL && left >= 16 && (KEYS == KEYS_PLAIN || at >= 0)) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int j = 0; j < PK; ++j) ptx::cp_async_16(kdst + (n * PK + j) * 512, kp + n * 8 * kst + j * 64);
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int j = 0; j < PV; ++j) ptx::cp_async_16(vdst + n * 4 * LINE + (((vch + 8 * j) ^ ((vkey + 4 * n) & 7)) << 4), vp + n * 4 * vst + j * 128);
                    return 0xffffu;
                }
                const int keys = (KEYS == KEYS_PLAIN || at >= 0) ? max(min(left, 16), 0) : 0;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int j = 0; j < PK; ++j) {
                        const bool ok = n * 8 + g < keys && (FULL || t + 4 * j < chunks);
                        ptx::cp_async_16(kdst + (n * PK + j) * 512, ok ? kp + n * 8 * kst + j * 64 : p.k, ok);
                    }
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int j = 0; j < PV; ++j) {
                        const bool ok = n * 4 + vkey < keys && (FULL || vch + 8 * j < chunks);
                        ptx::cp_async_16(vdst + n * 4 * LINE + (((vch + 8 * j) ^ ((vkey + 4 * n) & 7)) << 4), ok ? vp + n * 4 * vst + j * 128 : p.v, ok);
                    }
                return (1u << keys) - 1u;
            } else {
                const bool paged = p.table != nullptr;
                const long long ko = at < 0 ? -1 : paged ? ((at >> 32) * p.k_sb + static_cast<int>(at) * p.k_st) * 2 : at * kst;
                const long long vo = at < 0 ? -1 : paged ? ((at >> 32) * p.v_sb + static_cast<int>(at) * p.v_st) * 2 : at * vst;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const long long o = __shfl_sync(0xffffffffu, ko, n * 8 + g);
#pragma unroll
                    for (int j = 0; j < PK; ++j) {
                        const bool ok = o >= 0 && (FULL || t + 4 * j < chunks);
                        ptx::cp_async_16(kdst + (n * PK + j) * 512, ok ? kbase + o + j * 64 : p.k, ok);
                    }
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const long long o = __shfl_sync(0xffffffffu, vo, n * 4 + vkey);
#pragma unroll
                    for (int j = 0; j < PV; ++j) {
                        const bool ok = o >= 0 && (FULL || vch + 8 * j < chunks);
                        ptx::cp_async_16(vdst + n * 4 * LINE + (((vch + 8 * j) ^ ((vkey + 4 * n) & 7)) << 4), ok ? vbase + o + j * 128 : p.v, ok);
                    }
                }
                return __ballot_sync(0xffffffffu, at >= 0) & 0xffffu;
            }
        };
        unsigned kept[STAGES];  // which of a stage's 16 keys count
        long long next = ask(0);
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) {
            const long long at = next;
            next = ask(s + 1);
            kept[s] = 0u;
            if (s < n_units) kept[s] = fetch(s, s, at);
            ptx::cp_async_commit();
        }
        // ---------------------------------------------------------------- q: fragments of columns (queries) 8 nb + g
        uint32_t qf[NB][2 * PK][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < PK; ++j) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                const int r = nb * 8 + g, row = row0 + r;
                if (r < rows && (FULL || t + 4 * j < chunks)) {
                    const int tok = row / p.group, h = hk * p.group + row - tok * p.group;
                    w = *reinterpret_cast<const uint4*>(p.q + (b * p.q_sb + tok * p.q_st + h * p.q_sh + (t + 4 * j) * 8) * 2);
                }
                qf[nb][2 * j][0] = w.x, qf[nb][2 * j][1] = w.y, qf[nb][2 * j + 1][0] = w.z, qf[nb][2 * j + 1][1] = w.w;
            }
        float o[NB][DP / 16][4];
        float m[NB][2], l[NB][2];  // queries 8 nb + 2 t and + 1
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int x = 0; x < DP / 16; ++x) o[nb][x][0] = o[nb][x][1] = o[nb][x][2] = o[nb][x][3] = 0.0f;
            m[nb][0] = m[nb][1] = kLowest;
            l[nb][0] = l[nb][1] = 0.0f;
        }
        // ---------------------------------------------------------------- keys
        for (int i0 = 0; i0 < n_units; i0 += STAGES) {
#pragma unroll
            for (int s = 0; s < STAGES; ++s) {
                const int i = i0 + s;
                if (i < n_units) {
                    ptx::cp_async_wait<STAGES - 2>();
                    __syncwarp();  // the other lanes' copies too; and what is filled next has been read by every lane
                    {
                        constexpr int A = STAGES - 1;
                        const long long at = next;
                        next = ask(i + A + 1);
                        if (i + A < n_units) kept[(s + A) % STAGES] = fetch((s + A) % STAGES, i + A, at);
                        ptx::cp_async_commit();
                    }
                    const uint32_t st = ring + s * STAGE;
                    float sc[NB][4];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.0f;
#pragma unroll
                    for (int j = 0; j < PK; ++j) {
                        const uint4 lo = ptx::lds_128(st + lane * 16 + j * 512), hi = ptx::lds_128(st + lane * 16 + (PK + j) * 512);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            ptx::mma_16816<BF16>(sc[nb], lo.x, hi.x, lo.y, hi.y, qf[nb][2 * j][0], qf[nb][2 * j][1]);
                            ptx::mma_16816<BF16>(sc[nb], lo.z, hi.z, lo.w, hi.w, qf[nb][2 * j + 1][0], qf[nb][2 * j + 1][1]);
                        }
                    }
                    const unsigned kp = kept[s];
                    if (kp != 0xffffu) {
                        const bool lo = (kp >> g) & 1u, hi = (kp >> (8 + g)) & 1u;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            if (!lo) sc[nb][0] = sc[nb][1] = -INFINITY;
                            if (!hi) sc[nb][2] = sc[nb][3] = -INFINITY;
                        }
                    }
                    bool grew = false;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int r = 0; r < 2; ++r) grew |= fmaxf(sc[nb][r] - m[nb][r], sc[nb][2 + r] - m[nb][r]) * c > 8.0f;
                    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                float x = fmaxf(fmaxf(sc[nb][r], sc[nb][2 + r]), m[nb][r]);
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                                const float f = x == m[nb][r] ? 1.0f : ptx::exp2_approx((m[nb][r] - x) * c);
                                m[nb][r] = x;
                                l[nb][r] *= f;
#pragma unroll
                                for (int y = 0; y < DP / 16; ++y) {
                                    o[nb][y][r] *= f;
                                    o[nb][y][2 + r] *= f;
                                }
                            }
                    }
                    uint32_t ph[NB][2], pl[NB][2];  // P^T fragments: keys 0-7 and 8-15
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        float e[4];
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            e[r] = ptx::exp2_approx(fmaf(sc[nb][r] - m[nb][r], c, decode_lift<BF16>()));
                            e[2 + r] = ptx::exp2_approx(fmaf(sc[nb][2 + r] - m[nb][r], c, decode_lift<BF16>()));
                            l[nb][r] += e[r] + e[2 + r];
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t w = pack_16<BF16>(e[2 * h], e[2 * h + 1]);
                            const float2 f = unpack_16<BF16>(w);
                            ph[nb][h] = ptx::transposed_8x8(w);
                            pl[nb][h] = ptx::transposed_8x8(pack_16<BF16>(e[2 * h] - f.x, e[2 * h + 1] - f.y));
                        }
                    }
#pragma unroll
                    for (int x = 0; x < DP / 16; ++x) {
                        uint32_t v[4];
                        ptx::ldmatrix_x4_trans(st + vread + (((2 * x + mch) ^ (mkey & 7)) << 4), v);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            ptx::mma_16816<BF16>(o[nb][x], v[0], v[1], v[2], v[3], ph[nb][0], ph[nb][1]);
                            ptx::mma_16816<BF16>(o[nb][x], v[0], v[1], v[2], v[3], pl[nb][0], pl[nb][1]);
                        }
                    }
                }
            }
        }
        // ---------------------------------------------------------------- the four warps' results
        ptx::cp_async_wait<0>();
        __syncthreads();  // the rings are free: [warp][16 rows][DP + 4] sums, then [warp][16][2] maximum and sum
        float* sums = reinterpret_cast<float*>(smem_raw);
        float* stat = sums + kDecodeWarps * 16 * (DP + 4);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float s = l[nb][r];
                s += __shfl_xor_sync(0xffffffffu, s, 4);
                s += __shfl_xor_sync(0xffffffffu, s, 8);
                s += __shfl_xor_sync(0xffffffffu, s, 16);
                const int row = nb * 8 + 2 * t + r;
                if (row >= rows) continue;
                float* to = sums + (warp * 16 + row) * (DP + 4) + g;
#pragma unroll
                for (int x = 0; x < DP / 16; ++x) {
                    to[16 * x] = o[nb][x][r];
                    to[16 * x + 8] = o[nb][x][2 + r];
                }
                if (g == 0) {
                    stat[(warp * 16 + row) * 2] = m[nb][r];
                    stat[(warp * 16 + row) * 2 + 1] = s;
                }
            }
        __syncthreads();
        float* part = p.parts + static_cast<long long>(walk.slot()) * decode_slot(p.size);
        for (int id = threadIdx.x; id < rows * chunks; id += kDecodeThreads) {
            const int r = id / chunks, ch = id - r * chunks;
            float mm = kLowest, ll = 0.0f, f[kDecodeWarps], acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kDecodeWarps; ++w) mm = fmaxf(mm, stat[(w * 16 + r) * 2]);
#pragma unroll
            for (int w = 0; w < kDecodeWarps; ++w) {
                f[w] = ptx::exp2_approx((stat[(w * 16 + r) * 2] - mm) * c);
                ll += f[w] * stat[(w * 16 + r) * 2 + 1];
                const float* from = sums + (w * 16 + r) * (DP + 4) + ch * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] += f[w] * from[e];
            }
            if (whole) {
                const float inv = ll > 0.0f ? 1.0f / ll : (ll == 0.0f ? 0.0f : ll);  // no key kept: zeros; a NaN stays one
                const int row = row0 + r, tok = row / p.group, h = hk * p.group + row - tok * p.group;
                uint4 w;
                w.x = pack_16<BF16>(acc[0] * inv, acc[1] * inv);
                w.y = pack_16<BF16>(acc[2] * inv, acc[3] * inv);
                w.z = pack_16<BF16>(acc[4] * inv, acc[5] * inv);
                w.w = pack_16<BF16>(acc[6] * inv, acc[7] * inv);
                *reinterpret_cast<uint4*>(p.y + (b * p.y_sb + tok * p.y_st + h * p.y_sh + ch * 8) * 2) = w;
            } else {
                float* to = part + r * p.size + ch * 8;
                *reinterpret_cast<float4*>(to) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                *reinterpret_cast<float4*>(to + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
                if (ch == 0) {
                    part[16 * p.size + 2 * r] = mm;
                    part[16 * p.size + 2 * r + 1] = ll;
                }
            }
        }
        __syncthreads();  // before the rings are filled again
    }
    if (threadIdx.x == 0) p.cuts[blockIdx.x] = cut;
    if (bad_page) atomicOr(p.status, DEV_STATUS_BAD_PAGE);
}

// Joins the partial results of the (sequence, kv head, row block) that the end of CTA blockIdx.x's range cuts first. The CTA left word
// of it: looked up from the lengths by a block for each sequence and head, it took a batch's square (16384 sequences of 30 keys, 16
// heads: 10.3 ms in all, 1.33 so).
template <bool BF16>
__global__ void __launch_bounds__(128) attention_join_kernel(const __grid_constant__ DecodeParams p) {
    ptx::wait_for_dependencies();
    const int4 cut = p.cuts[blockIdx.x];
    const int b = cut.x, c0 = blockIdx.x, c1 = cut.w;
    if (b < 0) return;
    const int hk = cut.y / p.row_blocks, row0 = (cut.y - hk * p.row_blocks) * p.block_rows;
    const int rows = min(p.block_rows, p.tokens * p.group - row0), chunks = p.size / 4;
    const long long slot_floats = decode_slot(p.size);
    const float* first_part = p.parts + cut.z * slot_floats;
    for (int id = threadIdx.x; id < rows * chunks; id += blockDim.x) {
        const int r = id / chunks, ch = id - r * chunks;
        // a running maximum, so that a part's statistics and values are asked for together
        float mm = kLowest, ll = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int c = c0; c <= c1; ++c) {
            const float* part = c == c0 ? first_part : p.parts + 2ll * c * slot_floats;
            const float4 x = *reinterpret_cast<const float4*>(part + r * p.size + ch * 4);
            const float2 st = *reinterpret_cast<const float2*>(part + 16 * p.size + 2 * r);
            const float m_new = fmaxf(mm, st.x);
            const float f = ptx::exp2_approx((mm - m_new) * p.c), g = ptx::exp2_approx((st.x - m_new) * p.c);
            mm = m_new;
            ll = ll * f + st.y * g;
            acc[0] = acc[0] * f + x.x * g;
            acc[1] = acc[1] * f + x.y * g;
            acc[2] = acc[2] * f + x.z * g;
            acc[3] = acc[3] * f + x.w * g;
        }
        const float inv = ll > 0.0f ? 1.0f / ll : (ll == 0.0f ? 0.0f : ll);
        const int row = row0 + r, tok = row / p.group, h = hk * p.group + row - tok * p.group;
        uint2 w;
        w.x = pack_16<BF16>(acc[0] * inv, acc[1] * inv);
        w.y = pack_16<BF16>(acc[2] * inv, acc[3] * inv);
        *reinterpret_cast<uint2*>(p.y + (b * p.y_sb + tok * p.y_st + h * p.y_sh + ch * 4) * 2) = w;
    }
}

// New keys and values into a paged cache: token i of K and V to position positions[i] of sequence sequences[i] (null: i). Tokens
// whose sequence, position or page does not exist are left out and reported; those with positions below 0 are padding, left out. A thread moves 16 bytes; HBM-bound where there are
// many tokens, a launch's latency where there are few.
struct AppendParams {
    const char* k;
    const char* v;
    char* k_pages;
    char* v_pages;
    long long k_st, k_sh, v_st, v_sh;              // elements
    long long kp_sb, kp_st, kp_sh, vp_sb, vp_st, vp_sh;
    const int* table;
    long long table_sb;
    const int* positions;
    const int* sequences;
    int tokens, batch, table_width, page_size, num_pages, kv_heads, size;
    int* status;
};
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ AppendParams p) {
    ptx::launch_dependents();
    ptx::wait_for_dependencies();
    const int chunks = p.size / 8, per = p.kv_heads * chunks;
    const long long total = static_cast<long long>(p.tokens) * per;
    bool bad = false;
    for (long long id = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; id < total; id += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int tok = static_cast<int>(id / per), rest = static_cast<int>(id - static_cast<long long>(tok) * per);
        const int h = rest / chunks, ch = rest - h * chunks;
        const int pos = p.positions[tok], seq = p.sequences != nullptr ? p.sequences[tok] : tok;
        const int pg = pos / p.page_size, place = pos - pg * p.page_size;
        if (pos < 0) continue;  // padding
        if (seq < 0 || seq >= p.batch || pg >= p.table_width) {
            bad = true;
            continue;
        }
        const int page = p.table[seq * p.table_sb + pg];
        if (plan_place(page, place, p.num_pages) < 0) {
            bad = true;
            continue;
        }
        const uint4 k = *reinterpret_cast<const uint4*>(p.k + (tok * p.k_st + h * p.k_sh + ch * 8) * 2);
        const uint4 v = *reinterpret_cast<const uint4*>(p.v + (tok * p.v_st + h * p.v_sh + ch * 8) * 2);
        *reinterpret_cast<uint4*>(p.k_pages + (page * p.kp_sb + place * p.kp_st + h * p.kp_sh + ch * 8) * 2) = k;
        *reinterpret_cast<uint4*>(p.v_pages + (page * p.vp_sb + place * p.vp_st + h * p.vp_sh + ch * 8) * 2) = v;
    }
    if (bad) atomicOr(p.status, DEV_STATUS_BAD_PAGE);
}

}  // namespace dlfb200
