// paged_walk.h — which keys a tile's walk looks up where its rows see separate
// ranges of them (host and device code).
//
// A walk goes from the least key that a row sees to the largest.  Ranges that leave a gap between them cut what is
// seen into parts; a key in a gap has its table entry and row left alone, and the last seen key before
// it stands in for it (its weight is 0 in every row).  A part begins at a seen key behind one that is not
// seen and ends before the next that is not.
#pragma once

#ifdef __HIPCC__
#define IE_BOTH __host__ __device__ __forceinline__
#else
#define IE_BOTH inline
#endif

namespace ie {

// Keys lo <= j < hi of one row; lo >= hi is none.
struct KeyRange {
    int lo, hi;
};
// Whether `other` shows that no part begins where range `mine` does: it sees the key before, or begins at the same
// one and comes first (so that a part is found once).
IE_BOTH bool hides_begin(KeyRange mine, KeyRange other, bool first) {
    return other.lo < other.hi && (other.lo < mine.lo || (other.lo == mine.lo && first)) && other.hi >= mine.lo;
}
// The same for where it ends: `other` sees key mine.hi.
IE_BOTH bool hides_end(KeyRange mine, KeyRange other, bool first) {
    return other.lo < other.hi && (other.hi > mine.hi || (other.hi == mine.hi && first)) && other.lo <= mine.hi;
}
// Key p, or what stands in for it: begin and end are the largest of the parts' begins and ends up to p (end -1: none).
IE_BOTH int stand_in(int p, int begin, int end) { return end > begin ? end - 1 : p; }

}  // namespace ie
