// Host-side check of a strided output's rows.
#ifndef ROCWMMA_B200_CSRC_ROW_OVERLAP_H
#define ROCWMMA_B200_CSRC_ROW_OVERLAP_H

#include <cstdint>
#include <utility>

namespace b200wmma
{
    // Whether two of the rows of `length` elements at o * outerStride + i * innerStride, o < outer and
    // i < inner, share an element.
    inline bool rowsOverlap(uint64_t outer, uint64_t outerStride, uint64_t inner, uint64_t innerStride, uint64_t length)
    {
        if((outer > 1u && outerStride < length) || (inner > 1u && innerStride < length))
            return true;
        if(outer <= 1u || inner <= 1u)
            return false;
        if(outerStride < innerStride)
        {
            std::swap(outer, inner);
            std::swap(outerStride, innerStride);
        }
        // One block of rows behind the other: every usual layout.
        using Wide = unsigned __int128;
        if(outerStride >= Wide(innerStride) * (inner - 1u) + length)
            return false;
        // Blocks that reach into each other: the first row of each against its neighbours in the first
        // block.  (At most as many steps as the lesser of the two counts.)
        for(uint64_t o = 1; o < outer; ++o)
        {
            const Wide at = Wide(o) * outerStride, below = at / innerStride;
            if(below >= inner)
                return false;
            if(at - below * innerStride < length || (below + 1u < inner && (below + 1u) * innerStride - at < length))
                return true;
        }
        return false;
    }
} // namespace b200wmma
#endif
