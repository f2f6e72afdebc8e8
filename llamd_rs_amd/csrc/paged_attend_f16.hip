// paged_attend_f16.hip -- the paged attention (paged_attend.hpp) over f16 pages.
#include "paged_attend.hpp"

namespace llamd {

int launch_paged_attend_f16(const PagedAttendArgs &a, bool decode, hipStream_t st) {
    return paged_attend<ElemF16>(a, decode, st);
}

}  // namespace llamd
