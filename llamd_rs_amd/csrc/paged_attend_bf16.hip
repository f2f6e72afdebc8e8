// paged_attend_bf16.hip -- the paged attention (paged_attend.hpp) over bf16 pages.
#include "paged_attend.hpp"

namespace llamd {

int launch_paged_attend_bf16(const PagedAttendArgs &a, bool decode, hipStream_t st) {
    return paged_attend<ElemBF16>(a, decode, st);
}

}  // namespace llamd
