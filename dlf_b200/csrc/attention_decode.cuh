// Attention of few query rows over many keys: one new token (or a few) of each sequence over a paged cache or over an
// encoder's states.
//
//     y_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp2(c q_r.k_j - m_r),  c = scale * log2(e),  m_r the largest so far
//
// HBM-bound: the keys and values of a kv head are read once for up to 16 query rows (the query heads that share it), so
// what counts is how many bytes are in flight. A block has four warps; of a unit of 64 keys each takes 16 and runs the
// recurrence by itself (running maximum and sum, 32-bit accumulators), with its own ring of cp.async copies; the warps meet
// at the end of a segment (attention_plan.h). Products are mma.m16n8k16: 16 query rows, of which G are used.
//
// Every lane copies exactly the 16-byte pieces that its own fragments are made of, so a copy is followed by no barrier
// and read without bank conflicts (piece i of lane l lies at (32 i + l) * 16). With g = lane / 4, t = lane % 4:
//   K: lane (g, t) takes pieces t + 4 j of keys g and 8 + g. In q.k the head's d's may be taken in any order, so the four words
//      of a piece are the k-halves of two k-steps, and q's fragments are loaded in the same order.
//   V: lane (g, t) takes pieces g + 8 j of keys 2t, 2t+1, 2t+8, 2t+9 - the keys of its fragments - and pairs two keys'
//      words for each of the piece's eight d's; accumulator column n of n-tile (j, e) is then d = 8 (n + 8 j) + e.
// p is rounded to 16 bits for the second product in two parts (its rounding and the rest), which costs no time here and keeps
// the result as exact as 32-bit arithmetic.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_plan.h"
#include "ptx.cuh"

namespace dlfb200 {

enum : int { DEV_STATUS_BAD_PAGE = 2 };  // (bit 1 of the status word) a page table entry or a length beyond the cache

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
    int row_blocks;                                // blocks of 16 rows (row = token * group + head of the group)
    int ctas, least;
    float c;                                       // scale * log2(e)
    float* parts;                                  // slots of 16 x (size + 2) floats: sums, then maximum and sum of p per row
    int* status;
};

constexpr int kDecodeThreads = 128;
constexpr int kDecodeWarps = kDecodeThreads / 32;
DLF_HD constexpr int decode_stages(int dp) { return dp <= 64 ? 6 : 3; }
DLF_HD constexpr int decode_stage_bytes(int dp) { return 16 * dp * 2 * 2; }  // a warp's 16 keys and values
DLF_HD constexpr int decode_smem(int dp) { return kDecodeWarps * decode_stages(dp) * decode_stage_bytes(dp); }
DLF_HD constexpr int decode_slot(int size) { return 16 * (size + 2); }

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

// length of sequence b's keys; warp-uniform
__device__ __forceinline__ int decode_length(const DecodeParams& p, int b) {
    if (p.lengths == nullptr) return p.keys;
    bool bad = false;
    const int n = plan_length(p.lengths[b], p.keys, &bad);
    if (bad && threadIdx.x == 0) atomicOr(p.status, DEV_STATUS_BAD_PAGE);
    return n;
}

// units of all sequences for one (kv head, row block), and of those before sequence `upto`; by one warp
__device__ __forceinline__ void decode_units(const DecodeParams& p, int upto, long long& before, long long& all) {
    if (p.lengths == nullptr) {
        before = static_cast<long long>(upto) * plan_units(p.keys);
        all = static_cast<long long>(p.batch) * plan_units(p.keys);
        return;
    }
    const int lane = threadIdx.x & 31;
    int lo = 0, sum = 0;  // (host: all units fit in 31 bits)
    bool bad = false;
    for (int b = lane; b < p.batch; b += 32) {
        const int n = plan_units(plan_length(p.lengths[b], p.keys, &bad));
        sum += n;
        if (b < upto) lo += n;
    }
    before = __reduce_add_sync(0xffffffffu, lo);
    all = __reduce_add_sync(0xffffffffu, sum);
}

// the sequence that unit u of the call (u < all * heads) belongs to, and how many units lie before that sequence
__device__ __forceinline__ int decode_find(const DecodeParams& p, long long u, int heads, long long& before) {
    if (p.lengths == nullptr) {
        const long long n = static_cast<long long>(plan_units(p.keys)) * heads;
        const int b = static_cast<int>(u / n);
        before = b * n;
        return b;
    }
    const int lane = threadIdx.x & 31;
    long long sum = 0;
    bool bad = false;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int b = b0 + lane;
        const int n = b < p.batch ? plan_units(plan_length(p.lengths[b], p.keys, &bad)) : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, b < p.batch && u < (sum + incl) * heads);
        if (past) {
            const int src = __ffs(past) - 1;
            before = (sum + __shfl_sync(0xffffffffu, incl - n, src)) * heads;
            return b0 + src;
        }
        sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    before = sum * heads;
    return p.batch;
}

template <bool BF16, int DP, bool PAGED>
__global__ void __launch_bounds__(kDecodeThreads) attention_decode_kernel(const __grid_constant__ DecodeParams p) {
    constexpr int STAGES = decode_stages(DP);
    constexpr int PK = DP / 32;  // pieces of a key per lane (key g: t + 4 j, j < PK)
    constexpr int PV = DP / 64;  // pieces of a value per lane (g + 8 j, j < PV)
    constexpr int STAGE = decode_stage_bytes(DP);
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = ptx::smem_u32(smem_raw) + warp * STAGES * STAGE + lane * 16;

    ptx::launch_dependents();
    ptx::wait_for_dependencies();

    const int heads = p.kv_heads * p.row_blocks;
    long long before, all;
    decode_units(p, 0, before, all);
    all *= heads;
    const long long per = plan_per(all, p.ctas, p.least);
    long long u = blockIdx.x * per;
    const long long end = min(u + per, all);
    if (u >= end) return;
    int b = decode_find(p, u, heads, before);
    int len = decode_length(p, b);
    int units = plan_units(len);
    int hb = static_cast<int>((u - before) / units);       // head and row block
    int unit0 = static_cast<int>(u - before - static_cast<long long>(hb) * units);
    const int chunks = p.size / 8;
    bool bad_page = false;

    while (u < end) {
        const int n_units = static_cast<int>(min(static_cast<long long>(units - unit0), end - u));
        const bool whole = n_units == units;
        const int slot = plan_slot(u, per);
        const int hk = hb / p.row_blocks, row0 = (hb - hk * p.row_blocks) * 16;
        const int rows = min(16, p.tokens * p.group - row0);
        // ---------------------------------------------------------------- q
        uint32_t qf[2 * PK][4];
        auto q_piece = [&](int r, int j) -> uint4 {
            const int row = row0 + r, ch = t + 4 * j;
            if (r >= rows || ch >= chunks) return make_uint4(0u, 0u, 0u, 0u);
            const int tok = row / p.group, h = hk * p.group + row - tok * p.group;
            return *reinterpret_cast<const uint4*>(p.q + (b * p.q_sb + tok * p.q_st + h * p.q_sh + ch * 8) * 2);
        };
#pragma unroll
        for (int j = 0; j < PK; ++j) {
            const uint4 lo = q_piece(g, j), hi = q_piece(g + 8, j);
            qf[2 * j][0] = lo.x, qf[2 * j][1] = hi.x, qf[2 * j][2] = lo.y, qf[2 * j][3] = hi.y;
            qf[2 * j + 1][0] = lo.z, qf[2 * j + 1][1] = hi.z, qf[2 * j + 1][2] = lo.w, qf[2 * j + 1][3] = hi.w;
        }
        // ---------------------------------------------------------------- copies
        // step i of this warp: keys first_key + 64 i .. + 15 of the segment's units
        const int first_key = unit0 * kPlanUnit + warp * 16;
        const char* kbase = p.k + (PAGED ? 0 : b * p.k_sb * 2) + hk * p.k_sh * 2;
        const char* vbase = p.v + (PAGED ? 0 : b * p.v_sb * 2) + hk * p.v_sh * 2;
        const unsigned char* mask = p.mask != nullptr ? p.mask + b * p.mask_sb : nullptr;
        // lane l < 16 finds where key l of a step lies: its place in the cache (or its position), -1 = not kept
        auto find_row = [&](int i) -> long long {
            const int pos = first_key + i * kPlanUnit + (lane & 15);
            if (i >= n_units || pos >= len) return -1;
            if constexpr (PAGED) {
                const int pg = pos / p.page_size, place = pos - pg * p.page_size;
                const long long row = plan_place(p.table[b * p.table_sb + pg], place, p.num_pages);
                if (row < 0) bad_page = true;
                return row;
            } else {
                return mask != nullptr && mask[pos] == 0 ? -1 : pos;
            }
        };
        auto offset_of = [&](long long row, long long sb, long long st) -> long long {  // bytes
            if constexpr (PAGED) {
                return ((row >> 32) * sb + static_cast<int>(row) * st) * 2;
            } else {
                return row * st * 2;
            }
        };
        auto fetch = [&](int stage, long long row) {
            const uint32_t at = ring + stage * STAGE;
            const long long ko = row >= 0 ? offset_of(row, p.k_sb, p.k_st) : -1, vo = row >= 0 ? offset_of(row, p.v_sb, p.v_st) : -1;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const long long o = __shfl_sync(0xffffffffu, ko, n * 8 + g);
#pragma unroll
                for (int j = 0; j < PK; ++j) {
                    const bool ok = o >= 0 && t + 4 * j < chunks;
                    ptx::cp_async_16(at + (n * PK + j) * 512, kbase + (ok ? o + (t + 4 * j) * 16 : 0), ok);
                }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const long long o = __shfl_sync(0xffffffffu, vo, (n >> 1) * 8 + 2 * t + (n & 1));
#pragma unroll
                for (int j = 0; j < PV; ++j) {
                    const bool ok = o >= 0 && g + 8 * j < chunks;
                    ptx::cp_async_16(at + (2 * PK + n * PV + j) * 512, vbase + (ok ? o + (g + 8 * j) * 16 : 0), ok);
                }
            }
        };
        float o[8 * PV][4];
#pragma unroll
        for (int i = 0; i < 8 * PV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        unsigned kept[STAGES];  // which of a stage's 16 keys count
        long long next = find_row(0);
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) {
            const long long row = next;
            next = find_row(s + 1);
            kept[s] = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
            if (s < n_units) fetch(s, row);
            ptx::cp_async_commit();
        }
        // ---------------------------------------------------------------- keys
        for (int i0 = 0; i0 < n_units; i0 += STAGES) {
#pragma unroll
            for (int s = 0; s < STAGES; ++s) {
                const int i = i0 + s;
                if (i < n_units) {
                    {
                        constexpr int A = STAGES - 1;
                        const long long row = next;
                        next = find_row(i + A + 1);
                        kept[(s + A) % STAGES] = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
                        if (i + A < n_units) fetch((s + A) % STAGES, row);
                        ptx::cp_async_commit();
                    }
                    ptx::cp_async_wait<STAGES - 1>();
                    const uint32_t at = ring + s * STAGE;
                    float sc[2][4];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
#pragma unroll
                        for (int j = 0; j < PK; ++j) {
                            const uint4 kk = ptx::lds_128(at + (n * PK + j) * 512);
                            ptx::mma_16816<BF16>(sc[n], qf[2 * j][0], qf[2 * j][1], qf[2 * j][2], qf[2 * j][3], kk.x, kk.y);
                            ptx::mma_16816<BF16>(sc[n], qf[2 * j + 1][0], qf[2 * j + 1][1], qf[2 * j + 1][2], qf[2 * j + 1][3], kk.z, kk.w);
                        }
                    }
                    const unsigned kp = kept[s];
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool in = (kp >> (n * 8 + 2 * t + (e & 1))) & 1u;
                            sc[n][e] = in ? sc[n][e] * p.c : -INFINITY;
                            mx[e >> 1] = fmaxf(mx[e >> 1], sc[n][e]);
                        }
                    bool grew = false;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                        grew |= mx[r] > m[r];
                    }
                    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float m_new = fmaxf(m[r], mx[r]);
                            const float f = m_new == -INFINITY ? 1.0f : ptx::exp2_approx(m[r] - m_new);
                            m[r] = m_new;
                            l[r] *= f;
#pragma unroll
                            for (int x = 0; x < 8 * PV; ++x) {
                                o[x][2 * r] *= f;
                                o[x][2 * r + 1] *= f;
                            }
                        }
                    }
                    const float ms[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
                    uint32_t ph[4], pl[4];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float x = ptx::exp2_approx(sc[n][2 * r] - ms[r]), y = ptx::exp2_approx(sc[n][2 * r + 1] - ms[r]);
                            l[r] += x + y;
                            ph[n * 2 + r] = pack_16<BF16>(x, y);
                            const float2 h = unpack_16<BF16>(ph[n * 2 + r]);
                            pl[n * 2 + r] = pack_16<BF16>(x - h.x, y - h.y);
                        }
#pragma unroll
                    for (int j = 0; j < PV; ++j) {
                        const uint4 v0 = ptx::lds_128(at + (2 * PK + 0 * PV + j) * 512), v1 = ptx::lds_128(at + (2 * PK + 1 * PV + j) * 512);
                        const uint4 v2 = ptx::lds_128(at + (2 * PK + 2 * PV + j) * 512), v3 = ptx::lds_128(at + (2 * PK + 3 * PV + j) * 512);
                        const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
                        const uint32_t w2[4] = {v2.x, v2.y, v2.z, v2.w}, w3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
                            const uint32_t b0 = __byte_perm(w0[e >> 1], w1[e >> 1], sel), b1 = __byte_perm(w2[e >> 1], w3[e >> 1], sel);
                            ptx::mma_16816<BF16>(o[j * 8 + e], ph[0], ph[1], ph[2], ph[3], b0, b1);
                            ptx::mma_16816<BF16>(o[j * 8 + e], pl[0], pl[1], pl[2], pl[3], b0, b1);
                        }
                    }
                }
            }
        }
        // ---------------------------------------------------------------- the four warps' results
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        ptx::cp_async_wait<0>();
        __syncthreads();  // the rings are free: [warp][16 rows][DP + 4] sums, then [warp][16][2] maximum and sum
        float* sums = reinterpret_cast<float*>(smem_raw);
        float* stat = sums + kDecodeWarps * 16 * (DP + 4);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = g + 8 * r;
            if (row < rows) {
                float* to = sums + (warp * 16 + row) * (DP + 4);
#pragma unroll
                for (int j = 0; j < PV; ++j)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 8; e += 4)
                            *reinterpret_cast<float4*>(to + (2 * t + n + 8 * j) * 8 + e) =
                                make_float4(o[j * 8 + e][2 * r + n], o[j * 8 + e + 1][2 * r + n], o[j * 8 + e + 2][2 * r + n], o[j * 8 + e + 3][2 * r + n]);
                if (t == 0) {
                    stat[(warp * 16 + row) * 2] = m[r];
                    stat[(warp * 16 + row) * 2 + 1] = l[r];
                }
            }
        }
        __syncthreads();
        float* part = p.parts + static_cast<long long>(slot) * decode_slot(p.size);
        for (int id = threadIdx.x; id < rows * chunks; id += kDecodeThreads) {
            const int r = id / chunks, ch = id - r * chunks;
            float mm = -INFINITY, ll = 0.0f, f[kDecodeWarps], acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kDecodeWarps; ++w) mm = fmaxf(mm, stat[(w * 16 + r) * 2]);
#pragma unroll
            for (int w = 0; w < kDecodeWarps; ++w) {
                f[w] = mm == -INFINITY ? 0.0f : ptx::exp2_approx(stat[(w * 16 + r) * 2] - mm);
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
        // ---------------------------------------------------------------- next segment
        u += n_units;
        unit0 = 0;
        if (u < end && ++hb == heads) {
            hb = 0;
            ++b;
            len = decode_length(p, b);
            units = plan_units(len);
        }
    }
    if (bad_page) atomicOr(p.status, DEV_STATUS_BAD_PAGE);
}

// Joins the partial results of a (sequence, kv head, row block): a block each. Those that one CTA had whole are done already.
template <bool BF16>
__global__ void __launch_bounds__(128) attention_join_kernel(const __grid_constant__ DecodeParams p) {
    const int heads = p.kv_heads * p.row_blocks;
    const int b = blockIdx.x / heads, hb = blockIdx.x - b * heads;
    ptx::wait_for_dependencies();
    long long before, all;
    decode_units(p, b, before, all);
    const long long per = plan_per(all * heads, p.ctas, p.least);
    const int units = plan_units(decode_length(p, b));
    const long long first = before * heads + static_cast<long long>(hb) * units, last = first + units - 1;
    const int c0 = static_cast<int>(first / per), c1 = static_cast<int>(last / per);
    if (c0 == c1) return;
    const int hk = hb / p.row_blocks, row0 = (hb - hk * p.row_blocks) * 16;
    const int rows = min(16, p.tokens * p.group - row0), chunks = p.size / 4;
    const long long slot_floats = decode_slot(p.size);
    const float* first_part = p.parts + plan_slot(first, per) * slot_floats;
    for (int id = threadIdx.x; id < rows * chunks; id += blockDim.x) {
        const int r = id / chunks, ch = id - r * chunks;
        float mm = first_part[16 * p.size + 2 * r];
        for (int c = c0 + 1; c <= c1; ++c) mm = fmaxf(mm, p.parts[2ll * c * slot_floats + 16 * p.size + 2 * r]);
        float ll = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int c = c0; c <= c1; ++c) {
            const float* part = c == c0 ? first_part : p.parts + 2ll * c * slot_floats;
            const float f = mm == -INFINITY ? 0.0f : ptx::exp2_approx(part[16 * p.size + 2 * r] - mm);
            const float4 x = *reinterpret_cast<const float4*>(part + r * p.size + ch * 4);
            ll += f * part[16 * p.size + 2 * r + 1];
            acc[0] += f * x.x;
            acc[1] += f * x.y;
            acc[2] += f * x.z;
            acc[3] += f * x.w;
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
// whose sequence, position or page does not exist are left out and reported. A thread moves 16 bytes; HBM-bound where there are
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
        if (pos < 0 || seq < 0 || seq >= p.batch || pg >= p.table_width) {
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
