// piece.h -- V neighbouring values of a tensor in registers, as words: as an array
// of 16-bit values the compiler keeps each of them in a register of its own
// wherever it meets a branch.
#pragma once

#include <hip/hip_runtime.h>

namespace ssla {

template <class T, int V>
struct Piece {
    static constexpr bool kHalves = sizeof(T) == 2;
    static constexpr int kWords = (int)(sizeof(T) * V + 3) / 4;
    typedef T Pair __attribute__((ext_vector_type(2)));
    unsigned w[kWords];

    // At any alignment of the values'.
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kHalves && V == 1) w[0] = *(const unsigned short*)p;
        else __builtin_memcpy(w, p, sizeof(T) * V);
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kHalves && V == 1) *(unsigned short*)p = (unsigned short)w[0];
        else __builtin_memcpy(p, w, sizeof(T) * V);
    }
    // Values from the `over`-th on.
    __device__ __forceinline__ void store_from(T* p, int over) const {
        #pragma unroll
        for (int i = 1; i < V; ++i)
            if (i >= over) {
                if constexpr (kHalves) ((unsigned short*)p)[i] = (unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2]);
                else ((unsigned*)p)[i] = w[i];
            }
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (!kHalves) return __builtin_bit_cast(float, w[i]);
        else if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(float, i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else return (float)__builtin_bit_cast(Pair, w[i / 2])[i & 1];
    }
    // Rounded once.
    __device__ __forceinline__ void set(const float (&x)[V]) {
        #pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (!kHalves) w[i] = __builtin_bit_cast(unsigned, x[i]);
            else w[i] = __builtin_bit_cast(unsigned, Pair{(T)x[2 * i], 2 * i + 1 < V ? (T)x[2 * i + 1 < V ? 2 * i + 1 : 0] : (T)0.0f});
        }
    }
    __device__ __forceinline__ void zero() {
        #pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    // What the compiler has made of 16-bit values ends here: it would otherwise keep all
    // of them as floats from one use to the next.
    __device__ __forceinline__ void opaque() {
        if constexpr (kHalves) {
            #pragma unroll
            for (int i = 0; i < kWords; ++i) asm("" : "+v"(w[i]));
        }
    }
    // And here none of it has begun yet, behind a branch either.
    __device__ __forceinline__ void here() {
        if constexpr (kHalves) {
            #pragma unroll
            for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
        }
    }
};

}  // namespace ssla
