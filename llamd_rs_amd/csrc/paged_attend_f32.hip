// paged_attend_f32.hip -- the paged attention (paged_attend.hpp) over f32 pages.
#include "paged_attend.hpp"

namespace llamd {

int launch_paged_attend_f32(const PagedAttendArgs &a, bool decode, hipStream_t st) {
    return paged_attend<ElemF32>(a, decode, st);
}

}  // namespace llamd
