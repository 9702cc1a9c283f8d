// Attention over pools of signed 8-bit integers.
#include "attend_codes_launch.h"

namespace rch {

int launch_attend_int8(const rch_attend& A, int dtype, hipStream_t stream) {
    return launch_codes_rows<RCH_CODES_INT8>(A, dtype, stream);
}

}  // namespace rch
