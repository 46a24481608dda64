// linattn_f32.hip -- chunked linear attention over fp32 tokens (linattn_kernel.h).
#include "linattn_kernel.h"

namespace ssla {
hipError_t linattn_launch_f32(const LinAttnArgs& a, bool full, hipStream_t st) {
    return chunk::launch<float>(a, full, st);
}
}  // namespace ssla
