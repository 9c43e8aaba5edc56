// The count of asynchronous copies through a ring of slots, for the warp that starts them and waits for them.
#pragma once

#ifdef __CUDACC__
#define EXL3CU_HD __host__ __device__ __forceinline__
#else
#define EXL3CU_HD inline
#endif

namespace exl3cu {

// wait(slot, parity) waits for the slot's barrier to complete the phase of that parity, and is false when it has given
// up.  A copy that was not seen to land stays in flight: drain() waits for it once more, and for those behind it, before
// their memory is used for something else.
template <unsigned STAGES> struct CopyRing {
    unsigned landed = 0;
    // the slot of the copy `ahead` places behind the next one to land, STAGES - 1 at most
    EXL3CU_HD unsigned slot(unsigned ahead = 0) const { return (landed + ahead) % STAGES; }
    template <typename W> EXL3CU_HD bool next(W && wait) {
        if (!wait(slot(), landed / STAGES & 1u)) return false;
        ++landed;
        return true;
    }
    template <typename W> EXL3CU_HD void drain(int in_flight, W && wait) {
        for (; in_flight > 0; --in_flight, ++landed) (void)wait(slot(), landed / STAGES & 1u);
    }
};

}  // namespace exl3cu
