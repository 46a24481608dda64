// linattn_bf16.hip -- chunked linear attention over bf16 tokens (linattn_kernel.h).
#include "linattn_kernel.h"

namespace ssla {
hipError_t linattn_launch_bf16(const LinAttnArgs& a, bool full, hipStream_t st) {
    return chunk::launch<__bf16>(a, full, st);
}
}  // namespace ssla
