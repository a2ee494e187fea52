// Rows of 2 D bytes in LDS as operands of 16x16x32 matrix products: their places, their reads, the waits for direct loads.
#pragma once
#include "mdx_common.hpp"

namespace mdx {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const unsigned char*)p));
}

// Within a row the 16-byte pieces are exchanged by an exclusive or with the row (swizzle), so that 16 rows of one piece meet all
// banks once. The reads are inline asm that ends with its wait: the builtins would wait for every direct load in flight.
template <int D>
__device__ __forceinline__ int swizzle(int token) {  // exchanged piece = piece ^ swizzle(token)
    return D == 64 ? (token >> 1) & 7 : token & 15;
}
// tokens of half h: k-operands kk of the D / 32
template <int D>
__device__ __forceinline__ void read_k(u32x4 (&kf)[D / 32], uint32_t at) {
    if constexpr (D == 256) {
        asm volatile(
            "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
            "ds_read_b128 %4, %8 offset:256\n\tds_read_b128 %5, %9 offset:256\n\tds_read_b128 %6, %10 offset:256\n\t"
            "ds_read_b128 %7, %11 offset:256\n\ts_waitcnt lgkmcnt(0)"
            : "=&v"(kf[0]), "=&v"(kf[1]), "=&v"(kf[2]), "=&v"(kf[3]), "=&v"(kf[4]), "=&v"(kf[5]), "=&v"(kf[6]), "=&v"(kf[7])
            : "v"(at), "v"(at ^ 64), "v"(at ^ 128), "v"(at ^ 192)
            : "memory");
    } else if constexpr (D == 128) {
        asm volatile(
            "ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\tds_read_b128 %3, %7\n\ts_waitcnt lgkmcnt(0)"
            : "=&v"(kf[0]), "=&v"(kf[1]), "=&v"(kf[2]), "=&v"(kf[3])
            : "v"(at), "v"(at ^ 64), "v"(at ^ 128), "v"(at ^ 192)
            : "memory");
    } else {
        static_assert(D == 64, "head_dim 64, 128 or 256");
        asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(kf[0]), "=&v"(kf[1])
                     : "v"(at), "v"(at ^ 64)
                     : "memory");
    }
}
// what a wave may have in flight behind the load it waits for (vmcnt only)
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N <= 63, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace
}  // namespace mdx
