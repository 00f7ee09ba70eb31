// What the kernels that walk tiles with hand-ordered main loops share (block_product.hip, newton_schulz.hip): loops over constants, the barrier
// between stages, and which tile a workgroup takes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

namespace hiptk
{
    // f(integral_constant<int, 0>) ... f(integral_constant<int, N - 1>): what indexes registers must be a constant
    template <typename F, int... I>
    __device__ __forceinline__ void each_impl(F&& f, std::integer_sequence<int, I...>)
    {
        (f(std::integral_constant<int, I>{}), ...);
    }
    template <int N, typename F>
    __device__ __forceinline__ void each(F&& f)
    {
        each_impl(f, std::make_integer_sequence<int, N>{});
    }

    // A barrier that orders LDS alone (loads from memory stay under way across it)
    __device__ __forceinline__ void lds_barrier()
    {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    }

    // Place of workgroup wg in a list of `all` tiles of which the dies (XCDs: workgroup ids congruent mod 8, an L2 each) take contiguous ranges, so that an
    // L2 holds neighbours (X X^T of a batch of 12 x 1024 x 1024: 32 us with workgroups dealt round the dies, 24 us so)
    __device__ __forceinline__ uint32_t place_of(uint32_t wg, uint32_t all)
    {
        const uint32_t xcd = wg & 7, nth = wg >> 3, base = all >> 3, rem = all & 7;
        return xcd * base + (xcd < rem ? xcd : rem) + nth;
    }
    // Tile `lin` of a plane of tiles_p x tiles_q, walked in groups of 4 rows
    __device__ __forceinline__ void tile_of(uint32_t lin, int tiles_p, int tiles_q, int& tp, int& tq)
    {
        const uint32_t band = 4u * (uint32_t)tiles_q, g = lin / band, first = g * 4;
        const uint32_t rows = (uint32_t)tiles_p - first < 4 ? (uint32_t)tiles_p - first : 4, r = lin - g * band;
        tp                  = (int)(first + r % rows);
        tq                  = (int)(r / rows);
    }
}
