// ops_check.h -- what the checks of the sequence operators' C ABI share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "drain_scan.h"
#include "ssla_hip.h"

namespace ssla {

inline int refuse(const std::string& msg) {
    set_error(msg);
    return SSLA_ERR_ARG;
}

inline int hip_failed(const char* what, hipError_t e) {
    set_error(std::string(what) + ": " + hipGetErrorString(e));
    return SSLA_ERR_HIP;
}

inline bool is_dtype(int dtype) { return dtype == SSLA_F32 || dtype == SSLA_BF16 || dtype == SSLA_F16; }

inline size_t element(int dtype) { return dtype == SSLA_F32 ? 4 : 2; }

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Whether n0 x n1 pieces of `width` elements at strides s0, s1 are apart.
inline bool apart(long long n0, long long s0, long long n1, long long s1, long long width) {
    if (n0 <= 1) return n1 <= 1 || s1 >= width;
    if (n1 <= 1) return s0 >= width;
    if (s0 < s1) return s0 >= width && (s1 - width) / s0 >= n0 - 1;
    return s1 >= width && (s0 - width) / s1 >= n1 - 1;
}

// Whether a launch of a * b * c workgroups fits: HIP counts a grid's threads in 32 bits.
inline bool launchable(long long a, long long b, long long c, int threads) {
    return (__int128)a * b * c <= 0xffffffffll / threads;
}

// Kernels count tokens, rows and channels in 32 bits and step past the last one.
constexpr int kMaxCount = 0x7fff0000;
constexpr long long kMaxStride = 1ll << 40;      // offsets stay within 64 bits

inline bool is_stride(long long s) { return s >= 0 && s <= kMaxStride; }

}  // namespace ssla
