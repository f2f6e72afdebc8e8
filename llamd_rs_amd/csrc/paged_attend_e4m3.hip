// paged_attend_e4m3.hip -- the paged attention (paged_attend.hpp) over 8-bit pages.
#include "paged_attend.hpp"

namespace llamd {

int launch_paged_attend_e4m3(const PagedAttendArgs &a, bool decode, hipStream_t st) {
    return paged_attend<ElemE4M3>(a, decode, st);
}

}  // namespace llamd
