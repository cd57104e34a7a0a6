// Rows of the norms: how a part of a row is held, and its sums.
#pragma once

#include <type_traits>

#include "selective_common.h"

// Over the L lanes that share a part, 64 or the whole work-group; the same in all of them
template <int L>
__device__ __forceinline__ float norm_sum(float v, float* s) {
    v = sel_wave_sum(v);
    if constexpr (L > NHIP_WAVE) {
        const int wave = threadIdx.x / NHIP_WAVE;
        __syncthreads();
        if ((threadIdx.x & (NHIP_WAVE - 1)) == 0) s[wave] = v;
        __syncthreads();
        v = (s[0] + s[1]) + (s[2] + s[3]);
    }
    return v;
}

// How a part of `width` channels is held, `per16` of them side by side in a lane (one where rows do not allow
// wide reads): by a wave up to 128 times as many, by a group of four waves up to 1024 times; longer ones are read twice.
template <class F> static inline void norm_with_shape(bool vec, int per16, int width, F&& f) {
    const int v = vec ? per16 : 1;
    auto go = [&](auto lanes, auto held) {
        if (vec) f(std::true_type(), lanes, held);
        else f(std::false_type(), lanes, held);
    };
    using std::integral_constant;
    if (width <= 64 * v) go(integral_constant<int, 64>(), integral_constant<int, 1>());
    else if (width <= 128 * v) go(integral_constant<int, 64>(), integral_constant<int, 2>());
    else if (width <= 256 * v) go(integral_constant<int, 256>(), integral_constant<int, 1>());
    else if (width <= 512 * v) go(integral_constant<int, 256>(), integral_constant<int, 2>());
    else if (width <= 1024 * v) go(integral_constant<int, 256>(), integral_constant<int, 4>());
    else go(integral_constant<int, 256>(), integral_constant<int, 0>());
}

