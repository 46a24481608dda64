// linattn_bf16.hip -- chunked linear attention over bf16 tokens (linattn16.h).
#include "linattn16.h"

namespace ssla {
hipError_t linattn_launch_bf16(const LinAttnArgs& a, bool full, hipStream_t st) {
    return la16::launch<__bf16>(a, full, st);
}
}  // namespace ssla
