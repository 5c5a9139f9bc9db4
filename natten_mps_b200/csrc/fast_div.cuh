// Division of a non-negative 31-bit number by a divisor that is fixed for a launch: a product and a shift.
// n / d = (n * m) >> (31 + s) with s = ceil(log2 d), m = ceil(2^(31 + s) / d): m * d exceeds 2^(31 + s) by less than
// d <= 2^s, so the quotient is exact for n < 2^31 (Granlund and Montgomery, "Division by invariant integers using
// multiplication").
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace natten {

struct FastDiv {
    uint32_t d = 1, m = 0x80000000u, shift = 31;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor)
    {
        uint32_t s = 0;
        while (s < 31 && (1u << s) < divisor) ++s;
        shift = 31 + s;
        m = static_cast<uint32_t>(((1ull << shift) + divisor - 1) / divisor);
    }
    __host__ __device__ __forceinline__ int div(int n) const
    {
        return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * m) >> shift);
    }
    __host__ __device__ __forceinline__ int mod(int n, int q) const { return n - q * static_cast<int>(d); }
};

} // namespace natten
