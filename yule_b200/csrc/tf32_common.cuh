// tf32_common.cuh — fp32 products on the tensor core without fp32 operands: what the kernels for a batch served together (prefix_attention.cu, adapters.cu) share.
//
// An fp32 number is hi + lo, hi its upper 11 significant bits (a tf32 number, by truncation) and lo the exact rest, of which the tensor core keeps 11 bits again:
// a·b = hi·hi + hi·lo + lo·hi up to 2^-21 of |a·b|.  Truncation takes no number out of range, so unlike fp16 terms these need no scales: sizes of 1e-30 or 1e30
// beside one another keep their bits.
#pragma once

#include <cstdint>

namespace yule {
namespace {

// lo is made larger by 2^-11.5 of itself, a third to two thirds of its last place on the tensor core: in the mean nothing is cut off, and a lo of 11 bits comes out as it is.  Without it every
// product is short by 2.4e-7 of itself, which sums keep and soft-maxes multiply (error against 64 bits: attention 0.7e-6 to 1.0e-6, 0.4e-6 to 0.65e-6 so; adapters of ranks to 64 1.3e-7 to 7.6e-7,
// 1.0e-7 to 5.6e-7 so).
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
    hi = __float_as_uint(x) & 0xFFFFE000u;
    lo = __float_as_uint((x - __uint_as_float(hi)) * 1.000345f);
}
// d += a · b: 16×8 times 8×8.  With g = lane / 4, t = lane % 4: a0 (row g, column t), a1 (g + 8, t), a2 (g, t + 4), a3 (g + 8, t + 4); b0 (row t, column g), b1
// (t + 4, g); d0, d1 (row g, columns 2t, 2t + 1), d2, d3 (row g + 8).
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
}  // namespace
}  // namespace yule
