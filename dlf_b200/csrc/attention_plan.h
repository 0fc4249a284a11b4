// The arithmetic of how attention over many keys is shared out, in plain C++ (host and device) so that it can be tested
// without a GPU: where a key of a paged cache lies, and which part of which sequence a CTA takes.
//
// The work of a call is a row of units: for each sequence, for each of its `heads` (kv head, block of query rows), the
// sequence's units of kPlanUnit keys. A sequence without keys has one unit, in which its zeros are written. CTA c takes the units
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

constexpr int kPlanUnit = 64;

// a length as it comes from the caller: none below zero, none beyond what there is room for
DLF_HD int plan_length(int length, int most, bool* bad) {
    if (length > most) *bad = true;
    return length < 0 ? 0 : (length > most ? most : length);
}
DLF_HD int plan_units(int length) { return length <= 0 ? 1 : (length - 1) / kPlanUnit + 1; }

// units a CTA takes: at least `least`, below which a CTA's set-up and the joining cost more than they save
DLF_HD long long plan_per(long long total, int ctas, int least) {
    const long long per = (total + ctas - 1) / ctas;
    return per > least ? per : least;
}

DLF_HD int plan_slot(long long first_unit, long long per) {
    const long long c = first_unit / per;
    return static_cast<int>(2 * c + (first_unit == c * per ? 0 : 1));
}

// where a token of a paged cache lies, or -1 where the table's entry is no page of it
DLF_HD long long plan_place(int page, int place, int num_pages) {
    return page < 0 || page >= num_pages ? -1 : static_cast<long long>(page) << 32 | place;
}

}  // namespace dlfb200
