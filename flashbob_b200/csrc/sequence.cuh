// Ragged sequences in pages: lengths, new tokens and the page table, which only the GPU knows, and their checks.
#pragma once

#include <cstdint>

namespace bob {

enum : int { kStatusBadPage = 21, kStatusBadLength = 22 };

struct SequenceParams {
    const int* table; long long table_stride;      // null: page i of sequence b is page b * max_pages + i
    const int* lengths;
    const int* counts;            // null: every row of the call
    int B, max_pages, pages, page_shift, room;       // room: rows that a sequence has pages for
    int* sticky;                  // host-visible status word (may be null)
    int first;                    // least position of row 0: 0, or any negative number where the call's rows have no positions in the
                                  // sequence (attention without a causal mask) and may be more than it has
};

__device__ __forceinline__ void report(int* sticky, int code) {
    if (sticky) { *reinterpret_cast<volatile int*>(sticky) = code; __threadfence_system(); }
}

// start: position of row 0 (negative only where rows have none).  One that is not ok is empty: what its length and count would
// lead to belongs to nobody's call.
struct Sequence { int length, count, start; bool ok; };

__device__ __forceinline__ Sequence sequence_of(const SequenceParams& p, int b, int N) {
    Sequence s;
    const int length = __ldg(p.lengths + b), count = p.counts ? __ldg(p.counts + b) : N;
    s.ok = static_cast<unsigned>(length) <= static_cast<unsigned>(p.room) && static_cast<unsigned>(count) <= static_cast<unsigned>(N) &&
           length - count >= p.first;                        // (neither is above 2^28 here)
    s.length = s.ok ? length : 0;
    s.count = s.ok ? count : 0;
    s.start = s.length - s.count;
    return s;
}

// The table's entry for a position below its sequence's length, as it stands there.
__device__ __forceinline__ int page_entry(const SequenceParams& p, int b, int position) {
    if (!p.table) return b * p.max_pages + (position >> p.page_shift);
    return __ldg(p.table + b * p.table_stride + (position >> p.page_shift));
}

// ... -1 if it is no page.
__device__ __forceinline__ int page_of(const SequenceParams& p, int b, int position) {
    const int page = page_entry(p, b, position);
    return static_cast<unsigned>(page) < static_cast<unsigned>(p.pages) ? page : -1;
}

}  // namespace bob
