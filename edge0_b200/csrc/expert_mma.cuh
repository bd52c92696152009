// Building blocks of the tensor-core expert path: the NVFP4 -> fp16 decode, and the kernel that prepares expert-sorted fp16 activations.
// The instruction wrappers and descriptors are in tensor_core.cuh, the grouped GEMM itself is in expert_gemm.cuh.
//
// Parity mode: activations stay on the reference's int8 grid (q * d, exactly what the CPU path multiplies with).  The
// product q * d has up to 18 significant bits, so it is carried as TWO fp16 numbers hi + lo (exact for the fp16 block
// scales of Q8_0) and each K step issues the MMA twice into the same accumulator; NVFP4 weights (E2M1 value x UE4M3 block
// scale) are exact in fp16.  The MMA is kind::f16 with fp32 accumulation, so the result differs from the integer path
// only in fp32 summation order and in the tensor core's internal alignment of products (~3e-5 of RMS).  (A single fp16
// activation, 2^-12 relative, was measured at 3e-3 of RMS on `hidden` and pushed `down` past the 1e-2 bar through
// requantisation flips.)
//
// Operand roles are swapped with respect to the usual GEMM: D[feature, token] = W[feature, k] * A[token, k], so the
// fixed M = 128 of the instruction covers output features and N (16..128) covers however many rows an expert received.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "formats.cuh"
#include "router.cuh"
#include "tensor_core.cuh"

namespace b200moe {

// ---- activations for the tensor-core path --------------------------------------------------------------------------
// fp16(q * d) of the routed rows, gathered into expert order (row i of the output is routed row perm[i]) so every expert's
// rows are contiguous.  Within each group of 16 K positions the elements are stored in the order
// [0,8,1,9,2,10,3,11,4,12,5,13,6,14,7,15], the order in which the NVFP4 nibbles of a sub-block unpack.
// One warp per (sorted row, 32-element activation block).  Rows are row_stride halfs apart in both planes: K with the lo
// plane stored after the hi plane, 2K with out_lo = out_hi + K when hi and lo rows alternate.
__global__ void __launch_bounds__(256) sorted_act_fp16_kernel(ActQuant act, const int * perm, const int * meta, int rows,
                                                             int K, int n_ids, int ne11, __half * __restrict__ out_hi,
                                                             __half * __restrict__ out_lo, int row_stride) {
    pdl_wait();
    pdl_launch_dependents();

    const int warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    const int nb = K / 32;
    if (warp >= rows * nb) return;
    const int i = warp / nb, b = warp % nb;
    if (i >= meta[1]) return;   // rows that are in no group (empty exchange slots) have no sorted position
    const int r = perm[i];
    const int arow = (r / n_ids) * ne11 + (r % n_ids) % ne11;
    const float d = act.d[(size_t) arow * nb + b];
    const int q = act.q[(size_t) arow * K + b * 32 + lane];
    const int e = lane & 15;                                  // position inside the 16-group
    const int pos = (e < 8) ? 2 * e : 2 * (e - 8) + 1;        // 0->0, 8->1, 1->2, 9->3, ...
    const float v = __fmul_rn((float) q, d);
    const __half hi = __float2half_rn(v);
    const size_t o = (size_t) i * row_stride + b * 32 + (lane & 16) + pos;
    out_hi[o] = hi;
    out_lo[o] = __float2half_rn(__fsub_rn(v, __half2float(hi)));
}

struct MmaParams {
    const uint8_t * w0;     // [n_as][n_out][row_bytes] gate (DUAL) or the single tensor
    const uint8_t * w1;     // up (DUAL)
    const float * scale0;
    const float * scale1;
    const __half * act;     // [rows sorted by expert][K]  high part of q*d
    const __half * act_lo;  // same shape, low part
    const int * offsets;    // [n_as+1]
    const int * perm;       // [rows]
    const int * active;     // [n_as]
    const int * meta;
    float * out;            // [rows][n_out] indexed by routed row
    int n_out;
    int n_as;
    int * err;
};

// E2M1 magnitudes as the HIGH byte of their fp16 encoding: 0, .5, 1, 1.5 | 2, 3, 4, 6 (the low byte is zero for all of them)
constexpr uint32_t FP4_F16HI_LO = 0x3e3c3800u, FP4_F16HI_HI = 0x46444240u;

// 8 nibbles of one qs word -> 8 fp16 values (E2M1 value, signed) as four half2 words in the order
// [e0,e8] [e1,e9] [e2,e10] [e3,e11] (element j and j+8 of the sub-block share a byte).
__device__ __forceinline__ void fp4_word_to_half2x4(uint32_t w, uint32_t (&h)[4]) {
    const uint32_t wn = w ^ 0x88888888u;
    const uint32_t t = (w >> 3) & 0x11111111u;                       // sign of every nibble as 0/1
    // raw selector: positives give their byte, negatives give the replicated (zero) sign of the table byte
    const uint32_t a_lo = byte_perm(FP4_F16HI_LO, FP4_F16HI_HI, w), a_hi = byte_perm(FP4_F16HI_LO, FP4_F16HI_HI, w >> 16);
    const uint32_t c_lo = byte_perm(FP4_F16HI_LO, FP4_F16HI_HI, wn), c_hi = byte_perm(FP4_F16HI_LO, FP4_F16HI_HI, wn >> 16);
    const uint32_t s_lo = byte_perm(0x00008000u, 0u, t), s_hi = byte_perm(0x00008000u, 0u, t >> 16);
    const uint32_t b_lo = a_lo | c_lo | s_lo;                        // bytes: hi(e0) hi(e8) hi(e1) hi(e9)
    const uint32_t b_hi = a_hi | c_hi | s_hi;                        //        hi(e2) hi(e10) hi(e3) hi(e11)
    h[0] = byte_perm(b_lo, 0u, 0x1404);                              // [0, b0, 0, b1]
    h[1] = byte_perm(b_lo, 0u, 0x3424);
    h[2] = byte_perm(b_hi, 0u, 0x1404);
    h[3] = byte_perm(b_hi, 0u, 0x3424);
}

}  // namespace b200moe
