// The arithmetic of how attention over many keys is shared out, in plain C++ (host and device) so that it can be tested
// without a GPU: where a key of a paged cache lies, and which part of which sequence a CTA takes.
//
// The work of a call is a row of units: for each sequence, for each of its `heads` (head, block of query rows), the
// sequence's units of `unit` keys. A sequence without keys has one unit, in which its zeros are written. CTA c takes the units
// [c * per, (c + 1) * per): equal work whatever the lengths are. The part of a (sequence, head) that falls into a CTA's range is
// a segment. A segment that is all of it gives the result; any other gives a partial result in a slot of scratch memory,
// 2 c for the segment that starts a range and 2 c + 1 for a later one (which then ends the range, so there are no more), and
// the partial results of a (sequence, head) are joined in the order of the CTAs: the result does not depend on timing.
#pragma once

#ifdef __CUDACC__
#define DLF_HD __host__ __device__ __forceinline__
#else
#define DLF_HD inline
#endif

namespace dlfb200 {

// a length as it comes from the caller: none below zero, none beyond what there is room for
DLF_HD int plan_length(int length, int most, bool* bad) {
    if (length > most) *bad = true;
    return length < 0 ? 0 : (length > most ? most : length);
}
DLF_HD int plan_units(int length, int unit) { return length <= 0 ? 1 : (length - 1) / unit + 1; }

// units a CTA takes: at least `least`, below which a CTA's set-up and the joining cost more than they save
DLF_HD int plan_per(int total, int ctas, int least) {
    const int per = total / ctas + (total % ctas != 0);
    return per > least ? per : least;
}

DLF_HD int plan_slot(int first_unit, int per) {
    const int c = first_unit / per;
    return 2 * c + (first_unit == c * per ? 0 : 1);
}

// where a token of a paged cache lies, or -1 where the table's entry is no page of it
DLF_HD long long plan_place(int page, int place, int num_pages) {
    return page < 0 || page >= num_pages ? -1 : static_cast<long long>(page) << 32 | place;
}

#ifdef __CUDACC__
enum : int { DEV_STATUS_BAD_PAGE = 2 };  // (bit 1 of the status word) a page table entry or a length beyond the cache

struct PlanLengths {
    const int* lengths;  // or null: `keys` each
    int keys, batch, unit;
    int* status;
};

// what is the same in every lane, said so: the compiler then keeps it, and the branches and descriptors that depend on it, on the
// uniform datapath (the issue of a product otherwise takes as long as the product)
__device__ __forceinline__ int plan_uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ long long plan_uniform(long long x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ int plan_sequence(const PlanLengths& p, int b) {
    if (p.lengths == nullptr) return p.keys;
    bool bad = false;
    const int n = plan_length(p.lengths[b], p.keys, &bad);
    if (bad && threadIdx.x == 0) atomicOr(p.status, DEV_STATUS_BAD_PAGE);
    return plan_uniform(n);
}

// units of the sequences before `upto` and of all, for one head; by one warp
__device__ __forceinline__ void plan_sums(const PlanLengths& p, int upto, int& before, int& all) {
    if (p.lengths == nullptr) {
        before = upto * plan_units(p.keys, p.unit);
        all = p.batch * plan_units(p.keys, p.unit);
        return;
    }
    const int lane = threadIdx.x & 31;
    int lo = 0, sum = 0;
    bool bad = false;
    for (int b = lane; b < p.batch; b += 32) {
        const int n = plan_units(plan_length(p.lengths[b], p.keys, &bad), p.unit);
        sum += n;
        if (b < upto) lo += n;
    }
    before = __reduce_add_sync(0xffffffffu, lo);
    all = __reduce_add_sync(0xffffffffu, sum);
}

// the sequence that unit u of the call belongs to, and how many units lie before that sequence; by one warp
__device__ __forceinline__ int plan_find(const PlanLengths& p, int u, int heads, int& before) {
    if (p.lengths == nullptr) {
        const int n = plan_units(p.keys, p.unit) * heads;
        const int b = u / n;
        before = b * n;
        return b;
    }
    const int lane = threadIdx.x & 31;
    int sum = 0;
    bool bad = false;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int b = b0 + lane;
        const int n = b < p.batch ? plan_units(plan_length(p.lengths[b], p.keys, &bad), p.unit) : 0;
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

// A CTA's way through its units, segment by segment; every warp that needs it walks by itself.
struct PlanWalk {
    PlanLengths lengths;
    int u, end, per, heads;
    int b, head, unit0, units, len;  // the segment: sequence, head, first unit, units of the (sequence, head), keys

    __device__ __forceinline__ PlanWalk(const PlanLengths& l, int heads_, int ctas, int least) : lengths(l), heads(heads_) {
        int before, all;
        plan_sums(lengths, 0, before, all);
        all = plan_uniform(all) * heads;
        per = plan_per(all, ctas, least);
        u = static_cast<long long>(blockIdx.x) * per < all ? static_cast<int>(blockIdx.x) * per : all;
        end = per < all - u ? u + per : all;
        if (u >= end) return;
        b = plan_uniform(plan_find(lengths, u, heads, before));
        before = plan_uniform(before);
        len = plan_sequence(lengths, b);
        units = plan_units(len, lengths.unit);
        head = (u - before) / units;
        unit0 = u - before - head * units;
    }
    __device__ __forceinline__ bool more() const { return u < end; }
    __device__ __forceinline__ int count() const { return units - unit0 < end - u ? units - unit0 : end - u; }
    __device__ __forceinline__ bool whole() const { return count() == units; }
    __device__ __forceinline__ int slot() const { return plan_slot(u, per); }
    __device__ __forceinline__ void next() {
        u += count();
        unit0 = 0;
        if (u < end && ++head == heads) {
            head = 0;
            ++b;
            len = plan_sequence(lengths, b);
            units = plan_units(len, lengths.unit);
        }
    }
    // past sequences without keys
    __device__ __forceinline__ void next_with_keys() {
        do next();
        while (more() && len <= 0);
    }
};
#endif

}  // namespace dlfb200
