// linattn_f16.hip -- chunked linear attention over fp16 tokens (linattn_kernel.h).
#include "linattn_kernel.h"

namespace ssla {
hipError_t linattn_launch_f16(const LinAttnArgs& a, bool full, hipStream_t st) {
    return chunk::launch<_Float16>(a, full, st);
}
}  // namespace ssla
