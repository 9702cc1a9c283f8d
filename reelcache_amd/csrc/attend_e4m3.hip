// Attention over pools of 8-bit floats.
#include "attend_codes_launch.h"

namespace rch {

int launch_attend_e4m3(const rch_attend& A, int dtype, hipStream_t stream) {
    return launch_codes_rows<RCH_CODES_E4M3>(A, dtype, stream);
}

}  // namespace rch
