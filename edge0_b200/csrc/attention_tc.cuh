// Attention of many query rows to a key/value head (a shared prefix read by a whole batch, chunks of prompts) on tcgen05: 128 rows to a block,
// keys in tiles of 128 (head_dim 256: 64), scores and outputs in tensor memory.  The same contract as attend_kernel (attention.cuh) for
// bf16 queries; which of the two runs is decided by the rows (decoder_ops.cu).
//
// Roles, meeting at mbarriers (every wait is bounded; two stages of keys, values, scores and weights):
//   warps 0-7    softmax: a thread has half of the tile's keys of one row (a warp reads the 32 tensor-memory lanes of its rank in its warpgroup), takes the
//                maximum with its partner of the other half, writes the weights to tensor memory as f16, scales the outputs back when the
//                reference has to rise, and at the end reads them out
//   warps 8-15   producers: cache rows through registers into f16 operand tiles (128B swizzle), the next tile's loads in flight meanwhile
//   warp 16      one thread issues S = Q K^T (both operands from shared memory) and O += P V (P from tensor memory, V as it lies, head_dim contiguous)
//
// Precision.  Every operand is f16 and every factor a power of two or outside: rows of Q and of BF16 and Q4 caches are brought to the same size by a power of
// two a row (bf16's 8 bits, and a 3-bit code times an 8-bit scale, fit f16's 11), Q8 codes are whole numbers; a key's factor multiplies its score,
// a value's its weight, in fp32.  The weights 2^(s - ref) times the values' factors are rounded to f16 (2^-11).  ref rises only when a tile's
// maximum is more than 2^8 above it: weights stay below 2^15, sums are fp32.
//
// Bound by the issue of the softmax and the conversion: 128 x 128 scores cost about 6.5 instructions each, 32 K values about 1.2 (Q8), together 1,300 cycles
// of a scheduler, where the two products need 1,024 of the tensor pipe.
#pragma once
#include "attention.cuh"
#include "tensor_core.cuh"

namespace b200moe {

constexpr int TC_SOFTMAX_WARPS = 8, TC_PRODUCER_WARPS = 8;
constexpr int TC_THREADS = 32 * (TC_SOFTMAX_WARPS + TC_PRODUCER_WARPS + 1);
constexpr int TC_ROWS = 128;

template <int TYPE, int D>
struct TcShape {
    static constexpr int KT = D == 256 ? 64 : 128;                                     // keys to a tile
    static constexpr int VALUES = TYPE == KV_BF16 ? 8 : TYPE == KV_Q8 ? 16 : 32;       // of a row in a producer's 16 bytes
    static constexpr int TPR = D / VALUES;                                             // producers to a row
    static constexpr int ROWS = 32 * TC_PRODUCER_WARPS / TPR;                          // rows to a pass of all producers
    static constexpr int NL = KT / ROWS;                                               // passes
    static constexpr int Q_BYTES = TC_ROWS * D * 2, KV_BYTES = KT * D * 2;
    static constexpr uint32_t T_S = 0, T_O = 2 * KT, T_P = T_O + D;                    // tensor-memory columns: scores (2), outputs, weights (2)
    static constexpr size_t SMEM = Q_BYTES + 4 * KV_BYTES + 1024;
    static_assert(T_P + KT <= 512, "tensor memory");
    static_assert(ROWS * NL == KT, "tile");
};

// D[tmem] (+)= A[tmem, 16-bit pairs in a column] * B[smem desc]
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32 lanes x N columns, without a wait
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t * r) {
    static_assert(N == 16, "pieces of 16 columns");
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t * r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// byte offset of 16-byte piece `chunk` of row `row` in a tile of `rows` rows of head_dim f16 values: blocks of 64 values, 128 bytes a row, swizzled
__device__ __forceinline__ uint32_t tc_offset(int rows, int row, int chunk) {
    return (uint32_t) ((chunk >> 3) * rows * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// descriptor of a V tile as the product's second operand with head_dim contiguous: 8-key groups 1024 bytes apart, 64-value blocks `block` bytes
__device__ __forceinline__ uint64_t umma_desc_v(uint32_t smem_addr, uint32_t block) {
    uint64_t d = 0;
    d |= (uint64_t) ((smem_addr >> 4) & 0x3fff);
    d |= (uint64_t) (block >> 4) << 16;
    d |= (uint64_t) (1024 >> 4) << 32;
    d |= (uint64_t) 1 << 46;
    d |= (uint64_t) 2 << 61;
    return d;
}

// 2^(14 - e) for the largest exponent field e among a row's values, and the power that undoes it; kept where both are normal
__device__ __forceinline__ float row_up(uint32_t amax_bits) {
    const int e = min(max((int) (amax_bits >> 23), 40), 250);
    return __uint_as_float((uint32_t) (254 + 14 - e) << 23);
}
__device__ __forceinline__ float pow2_inverse(float p) { return __uint_as_float((254u << 23) - __float_as_uint(p)); }

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// what a producer holds of a tile: 16 bytes of each of its rows, and the row's scales
template <int TYPE, int D>
struct TcPiece {
    uint4 v[TcShape<TYPE, D>::NL];
    uint32_t s[TYPE == KV_BF16 ? 1 : TcShape<TYPE, D>::NL][TYPE == KV_Q4 ? D / 64 : 1];
};

template <int TYPE, int D>
__device__ __forceinline__ void tc_load(TcPiece<TYPE, D> & t, const uint8_t * rows, const void * scales, const int64_t * row, int x) {
    typedef TcShape<TYPE, D> S;
#pragma unroll
    for (int n = 0; n < S::NL; ++n) {
        t.v[n] = make_uint4(0, 0, 0, 0);
        if (row[n] >= 0) t.v[n] = load_stream(reinterpret_cast<const uint4 *>(rows + row[n] * kv_row_bytes<TYPE, D>() + 16 * x));
        if (TYPE == KV_Q8) t.s[n][0] = row[n] >= 0 ? static_cast<const uint32_t *>(scales)[row[n]] : 0u;
        if (TYPE == KV_Q4)
#pragma unroll
            for (int g = 0; g < D / 64; ++g) t.s[n][g] = row[n] >= 0 ? static_cast<const uint32_t *>(scales)[row[n] * (D / 64) + g] : 0u;
    }
}

// converts a row's 16 bytes and stores them; returns the row's factor.  clean: values that are not finite are stored as zeros and the factor is NaN.
template <int TYPE, int D, bool VALUES>
__device__ __forceinline__ float tc_store(const TcPiece<TYPE, D> & t, int n, uint8_t * tile, int row, int x, bool there, bool clean) {
    typedef TcShape<TYPE, D> S;
    if (TYPE == KV_Q8) {
        uint4 lo, hi;
        const uint32_t w[4] = { t.v[n].x, t.v[n].y, t.v[n].z, t.v[n].w };
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[2 * i] = there ? bytes_to_half2(w[i], 0x4140) : 0u;
            h[2 * i + 1] = there ? bytes_to_half2(w[i], 0x4342) : 0u;
        }
        lo = make_uint4(h[0], h[1], h[2], h[3]);
        hi = make_uint4(h[4], h[5], h[6], h[7]);
        // the threads of a row's second 64 values begin with the other piece: their block lies on the same banks
        const int first = (x >> 2) & 1;
        *reinterpret_cast<uint4 *>(tile + tc_offset(S::KT, row, 2 * x + first)) = first ? hi : lo;
        *reinterpret_cast<uint4 *>(tile + tc_offset(S::KT, row, 2 * x + 1 - first)) = first ? lo : hi;
        return __uint_as_float(t.s[n][0]);
    } else if (TYPE == KV_Q4) {
        constexpr int GB = D >= 128 ? 4 : 2;
        constexpr int G = D / 32;
        // the scales brought below 2^12 by the largest one's exponent, so that a code's product stays below 2^15
        uint32_t top = 0;
        bool finite = true;
        uint32_t d[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            d[g] = g & 1 ? t.s[n][g / 2] & 0xffff0000u : t.s[n][g / 2] << 16;
            const bool ok = d[g] < 0x7f800000u;
            finite &= ok;
            if (ok) top = max(top, d[g]);
        }
        const float up = row_up(top) * 0.125f;
        const int run = x / (D >= 128 ? 4 : 2), in_run = D >= 128 ? x % 4 : x;
        const uint32_t w[4] = { t.v[n].x, t.v[n].y, t.v[n].z, t.v[n].w };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int g, c;
            uint32_t q;
            if (VALUES) {
                if (GB == 4) { g = i; c = in_run; q = __byte_perm(w[g / 2], w[2 + g / 2], g & 1 ? 0x7632 : 0x5410); }
                else { g = i & 1; c = 2 * in_run + (i >> 1); q = __byte_perm(w[2 * (i >> 1)], w[2 * (i >> 1) + 1], g ? 0x7632 : 0x5410); }
            } else {
                if (GB == 4) { g = i; c = in_run; q = w[i]; }
                else { g = i & 1; c = 2 * in_run + (i >> 1); q = w[i]; }
            }
            float scale = 0.0f;
#pragma unroll
            for (int j = 0; j < G; ++j) if (j == run * GB + g) scale = __uint_as_float(d[j]);
            const bool zero = !there || (clean && !(scale < INFINITY));
            const __half2 s2 = __float2half2_rn(scale * up);
            const uint32_t even = q & 0x0f0f0f0fu, odd = (q >> 4) & 0x0f0f0f0fu;
            const uint32_t a = __byte_perm(even, odd, 0x5140), b = __byte_perm(even, odd, 0x7362);    // nibbles 0 1 2 3, 4 5 6 7
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t u = __byte_perm(j < 2 ? a : b, 0x64646464u, j & 1 ? 0x4342 : 0x4140);
                const __half2 v = __hmul2(__hsub2(*reinterpret_cast<const __half2 *>(&u), __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408))), s2);
                h[j] = zero ? 0u : half2_bits(v);
            }
            *reinterpret_cast<uint4 *>(tile + tc_offset(S::KT, row, 4 * (run * GB + g) + c)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        return clean && !finite ? __uint_as_float(0x7fffffffu) : pow2_inverse(up);
    } else {
        const uint32_t w[4] = { t.v[n].x, t.v[n].y, t.v[n].z, t.v[n].w };
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
#pragma unroll
        for (int o = S::TPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float up = row_up(top);
        const bool zero = clean && top >= 0x7f800000u;    // the whole row: its weights become NaN
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            h[i] = zero ? 0u : half2_bits(__floats2half2_rn(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up));
        *reinterpret_cast<uint4 *>(tile + tc_offset(S::KT, row, x)) = make_uint4(h[0], h[1], h[2], h[3]);
        return zero ? __uint_as_float(0x7fffffffu) : pow2_inverse(up);
    }
}

template <int TYPE, int D, bool PREFIX>
__global__ void __launch_bounds__(TC_THREADS, 1) attend_tc_kernel(const __grid_constant__ AttnParams p) {
    typedef TcShape<TYPE, D> S;
    constexpr int KT = S::KT, HALF = KT / 2;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t * sq = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t) 1023);
    uint8_t * sk = sq + S::Q_BYTES, * sv = sk + 2 * S::KV_BYTES;
    __shared__ uint64_t k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], s_free[2], p_full[2], pv_done[2], met[4];
    __shared__ __align__(16) float k_scale[2][KT], v_scale[2][KT];
    __shared__ float2 other[2][2][TC_ROWS];    // what the two threads of a row tell one another
    __shared__ float s_factor[TC_ROWS];
    __shared__ int s_bad[2];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int at = blockIdx.x;
    const int row_tile = at % p.row_tiles;
    at /= p.row_tiles;
    const int head = at % p.kv.n_head;
    at /= p.kv.n_head;
    const int chunk = PREFIX ? at : at % p.own_chunks;
    const int seq = PREFIX ? 0 : at / p.own_chunks;
    int first = 0, n_new, len;
    const int front = PREFIX ? p.prefix_len : p.own_prefix;    // keys that every row sees, in the prefix's pages
    if (PREFIX) {
        n_new = min(max(p.q_start ? p.q_start[p.n_seq] : p.n_seq, 0), p.n_tokens);
        len = 0;
    } else if (!attn_sequence(p, seq, first, n_new, len, tid == 0 && row_tile == 0 && head == 0 && chunk == 0)) {
        return;
    }
    const int row0 = row_tile * TC_ROWS, n_rows = min(n_new * p.group - row0, TC_ROWS);
    const int per_chunk = PREFIX ? p.prefix_chunk : p.own_chunk, key0 = chunk * per_chunk;
    if (n_rows <= 0 || (key0 >= front + len && !(key0 == 0 && p.direct))) return;
    auto reach = [&](int row) { return PREFIX ? front : front + max(0, len - n_new + (row0 + row) / p.group + 1); };
    const int key_end = min(key0 + per_chunk, reach(n_rows - 1)), seen_by_all = reach(0);
    const int n_tiles = key_end > key0 ? (key_end - key0 + KT - 1) / KT : 0;
    // some row does not see all keys of the tile (rows behind n_rows are nobody's)
    auto masked_tile = [&](int i) { return key0 + (i + 1) * KT > min(seen_by_all, key_end); };

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 32 * TC_PRODUCER_WARPS);
            mbar_init(&v_full[i], 32 * TC_PRODUCER_WARPS);
            mbar_init(&k_free[i], 1 + TC_SOFTMAX_WARPS);
            mbar_init(&v_free[i], 1 + TC_SOFTMAX_WARPS);
            mbar_init(&s_full[i], 1);
            mbar_init(&s_free[i], 32 * TC_SOFTMAX_WARPS);
            mbar_init(&p_full[i], 32 * TC_SOFTMAX_WARPS);
            mbar_init(&pv_done[i], 1);
            s_bad[i] = 0;
        }
        for (int i = 0; i < 4; ++i) mbar_init(&met[i], 2);
        mbar_fence_init();
        s_abort = 0;
    }
    if (warp == TC_SOFTMAX_WARPS + TC_PRODUCER_WARPS) {
        tmem_alloc(&s_tmem, 512);
        tmem_relinquish();
    }
    // ---- the queries: D / 8 threads to a row
    {
        constexpr int TPR = D / 8, PASS = 32 * (TC_SOFTMAX_WARPS + TC_PRODUCER_WARPS) / TPR;
        const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
        if (warp < TC_SOFTMAX_WARPS + TC_PRODUCER_WARPS) {
#pragma unroll
            for (int r0 = 0; r0 < TC_ROWS; r0 += PASS) {
                const int row = r0 + tid / TPR, x = tid % TPR;
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.0f;
                if (row < n_rows) {
                    const int token = first + (row0 + row) / p.group, h = head * p.group + (row0 + row) % p.group;
                    load8<__nv_bfloat16>(v, p.q + (int64_t) token * p.q_token + (int64_t) h * p.q_head, x, p.q_aligned);
                }
                float most = 0.0f;    // NaN says nothing about the size
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
#pragma unroll
                for (int o = TPR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float up = row_up(__float_as_uint(most));
                uint32_t h2[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) h2[i] = half2_bits(__floats2half2_rn(v[2 * i] * (up * sign), v[2 * i + 1] * (up * sign)));
                *reinterpret_cast<uint4 *>(sq + tc_offset(TC_ROWS, row, x)) = make_uint4(h2[0], h2[1], h2[2], h2[3]);
                if (x == 0) s_factor[row] = fabsf(p.scale_log2) * pow2_inverse(up);
            }
        }
        fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp < TC_SOFTMAX_WARPS) {
        // ------------------------------------------------------------ softmax
        const int row = (warp & 3) * 32 + lane, half = warp >> 2;
        const uint32_t t_lane = tmem + ((uint32_t) ((warp & 3) * 32) << 16);
        const float factor = s_factor[row];
        const int seen = reach(min(row, n_rows - 1));
        float ref = -INFINITY, sum = 0.0f;
        bool ok = true;
        for (int i = 0; i < n_tiles; ++i) {
            const int st = i & 1;
            const uint32_t ph = (i >> 1) & 1;
            // the votes reconverge the warp and make the outcome uniform for the instructions that need all of it
            ok = __all_sync(0xffffffffu, wait_or_abort(&s_full[st], ph, &s_abort, p.err) && wait_or_abort(&k_full[st], ph, &s_abort, p.err));
            if (!ok) break;
            tc_fence_after();
            uint32_t s[HALF];
#pragma unroll
            for (int c = 0; c < HALF; c += 16) tmem_load<16>(t_lane + S::T_S + st * KT + half * HALF + c, s + c);
            tmem_wait_ld();
            tc_fence_before();
            mbar_arrive(&s_free[st]);
            const bool masked = masked_tile(i) || s_bad[st] == i + 1;
            const int key = key0 + i * KT + half * HALF;
            const float4 * ks = reinterpret_cast<const float4 *>(k_scale[st] + half * HALF);
            float most = -INFINITY;
#pragma unroll
            for (int c = 0; c < HALF; c += 4) {
                const float4 f = ks[c / 4];
                const float ff[4] = { f.x, f.y, f.z, f.w };
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float v = __uint_as_float(s[c + j]) * ff[j];
                    s[c + j] = __float_as_uint(v);
                    if (!masked) most = fmaxf(most, v);
                }
            }
            uint64_t on = ~0ull;    // keys that the row sees
            if (masked) {
                on = 0;
#pragma unroll
                for (int c = 0; c < HALF; ++c) {
                    // a negative factor marks a page that is not there
                    const bool see = key + c < seen && !(k_scale[st][half * HALF + c] < 0.0f);
                    if (see) { on |= 1ull << c; most = fmaxf(most, __uint_as_float(s[c])); }
                }
            }
            ok = __all_sync(0xffffffffu, wait_or_abort(&v_full[st], ph, &s_abort, p.err));    // the values' factors
            if (!ok) break;
            if (lane == 0) mbar_arrive(&k_free[st]);
            float top = 0.0f;    // the largest of the values' factors
            if (!masked) {
#pragma unroll
                for (int c = lane; c < KT; c += 32) top = fmaxf(top, v_scale[st][c]);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            } else {
#pragma unroll
                for (int c = 0; c < HALF; ++c) if (on >> c & 1) top = fmaxf(top, v_scale[st][half * HALF + c]);
            }
            other[st][half][row] = make_float2(most, top);
            __syncwarp();
            if (lane == 0) mbar_arrive(&met[warp & 3]);
            ok = __all_sync(0xffffffffu, wait_or_abort(&met[warp & 3], i & 1, &s_abort, p.err));
            if (!ok) break;
            const float2 partner = other[st][half ^ 1][row];
            most = fmaxf(most, partner.x);
            top = fmaxf(top, partner.y);
            // weights 2^(s - ref) times a factor stay below 2^7 at this reference, and below 2^15 until it has to rise
            const int e = max((int) (__float_as_uint(top) >> 23), 47);
            const float want = most == -INFINITY ? -INFINITY : most * factor + (float) (e - 127 - 6);
            const bool rise = want > ref + 8.0f || (ref == -INFINITY && want > -INFINITY);
            if (__any_sync(0xffffffffu, rise)) {
                const float back = !rise ? 1.0f : ref == -INFINITY ? 0.0f : fast_exp2(ref - want);
                if (rise) { sum *= back; ref = want; }
                if (i > 0) {
                    ok = __all_sync(0xffffffffu, wait_or_abort(&pv_done[st ^ 1], ((i - 1) >> 1) & 1, &s_abort, p.err));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < D / 2; c += 16) {
                        uint32_t o[16];
                        tmem_load<16>(t_lane + S::T_O + half * (D / 2) + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * back);
                        tmem_store16(t_lane + S::T_O + half * (D / 2) + c, o);
                    }
                    tmem_wait_st();
                }
            }
            const float base = ref == -INFINITY ? 0.0f : ref;
            const float4 * vs = reinterpret_cast<const float4 *>(v_scale[st] + half * HALF);
            uint32_t w[HALF / 2];
#pragma unroll
            for (int c = 0; c < HALF; c += 4) {
                const float4 f = vs[c / 4];
                const float ff[4] = { f.x, f.y, f.z, f.w };
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float e2 = fast_exp2(fmaf(__uint_as_float(s[c + j]), factor, -base));
                    x[j] = e2 * ff[j];
                    if (masked && !(on >> (c + j) & 1)) { e2 = 0.0f; x[j] = 0.0f; }
                    sum += e2;
                }
                w[c / 2] = half2_bits(__floats2half2_rn(x[0], x[1]));
                w[c / 2 + 1] = half2_bits(__floats2half2_rn(x[2], x[3]));
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_free[st]);
            // the weights' columns are free once the product two tiles back has read them
            ok = __all_sync(0xffffffffu, wait_or_abort(&pv_done[st], ph ^ 1u, &s_abort, p.err));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HALF / 2; c += 16) tmem_store16(t_lane + S::T_P + st * (KT / 2) + half * (HALF / 2) + c, w + c);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[st]);
        }
        // ---- the outputs
        if (ok && n_tiles) ok = __all_sync(0xffffffffu, wait_or_abort(&pv_done[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1, &s_abort, p.err));
        tc_fence_after();
        other[n_tiles & 1][half][row] = make_float2(sum, 0.0f);
        __syncwarp();
        if (lane == 0) mbar_arrive(&met[warp & 3]);
        if (ok) ok = __all_sync(0xffffffffu, wait_or_abort(&met[warp & 3], n_tiles & 1, &s_abort, p.err));
        if (ok) {
            sum += other[n_tiles & 1][half ^ 1][row].x;
            const int token = first + (row0 + row) / p.group, h = head * p.group + (row0 + row) % p.group;
            const int64_t line = (int64_t) token * p.n_head + h;
            const int chunks = p.prefix_chunks + p.own_chunks, slot = PREFIX ? chunk : p.prefix_chunks + chunk;
            const float inv = p.direct ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
            const bool there = row < n_rows;
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
                uint32_t o[16];
                if (n_tiles) {
                    tmem_load<16>(t_lane + S::T_O + half * (D / 2) + c, o);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = 0u;
                }
                const int d = half * (D / 2) + c;
                if (there && p.direct) {
                    float x[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = sum == 0.0f ? 0.0f : __uint_as_float(o[j]) * inv;
                    char * dst = p.out + (int64_t) token * p.out_token + (int64_t) h * p.out_head;
                    float lo[8], hi[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) { lo[j] = x[j]; hi[j] = x[8 + j]; }
                    store8<__nv_bfloat16>(lo, dst, d / 8, p.out_aligned);
                    store8<__nv_bfloat16>(hi, dst, d / 8 + 1, p.out_aligned);
                } else if (there) {
                    float4 * dst = reinterpret_cast<float4 *>(p.part_o + (line * chunks + slot) * D + d);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        dst[j] = make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]), __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3]));
                }
            }
            if (there && half == 0) {
                if (!p.direct) p.part_ml[line * chunks + slot] = make_float2(ref, sum);
                else if (p.lse) p.lse[line] = sum == 0.0f ? -INFINITY : (ref + log2f(sum)) * 0.69314718055994531f;
            }
        }
    } else if (warp < TC_SOFTMAX_WARPS + TC_PRODUCER_WARPS) {
        // ------------------------------------------------------------ producers
        const int q = tid - 32 * TC_SOFTMAX_WARPS, x = q % S::TPR, r0 = q / S::TPR;
        const int32_t * table = PREFIX ? p.prefix_pages : p.pages + (int64_t) seq * p.pages_stride;
        const int shift = p.kv.page_shift, in_page = (1 << shift) - 1, n_pages = (int) (p.kv.n_slots >> shift);
        int64_t row[S::NL];    // cache row of each pass, -1 behind the last key, -2 where the page is not there
        auto find = [&](int i) {
#pragma unroll
            for (int n = 0; n < S::NL; ++n) {
                const int key = key0 + i * KT + n * S::ROWS + r0;
                row[n] = -1;
                if (key >= key_end) continue;
                const bool shared = key < front;
                const int k = shared ? key : key - front;
                const int page = shared ? p.prefix_pages[k >> shift] : table[k >> shift];
                if (page < 0 || page >= n_pages) {
                    report_error(p.err, DEV_ERR_BAD_SLOT);
                    row[n] = -2;
                } else {
                    row[n] = (((int64_t) page * p.kv.n_head + head) << shift) + (k & in_page);
                }
            }
        };
        TcPiece<TYPE, D> k, v;
        uint32_t there = 0, gone = 0;    // of the tile whose values are held
        auto flags = [&]() {
            there = gone = 0;
#pragma unroll
            for (int n = 0; n < S::NL; ++n) {
                if (row[n] >= 0) there |= 1u << n;
                if (row[n] == -2) gone |= 1u << n;
            }
        };
        if (n_tiles) {
            find(0);
            tc_load<TYPE, D>(k, p.kv.k, p.kv.k_scale, row, x);
            tc_load<TYPE, D>(v, p.kv.v, p.kv.v_scale, row, x);
        }
        for (int i = 0; i < n_tiles; ++i) {
            const int st = i & 1;
            const uint32_t ph = (i >> 1) & 1;
            flags();
            const bool masked = masked_tile(i);
            if (!__all_sync(0xffffffffu, wait_or_abort<20>(&k_free[st], ph ^ 1u, &s_abort, p.err))) break;
#pragma unroll
            for (int n = 0; n < S::NL; ++n) {
                const float f = tc_store<TYPE, D, false>(k, n, sk + st * S::KV_BYTES, n * S::ROWS + r0, x, there >> n & 1, false);
                if (x == 0) k_scale[st][n * S::ROWS + r0] = gone >> n & 1 ? -1.0f : there >> n & 1 ? f : 0.0f;
            }
            if (gone) s_bad[st] = i + 1;
            fence_async_smem();
            mbar_arrive(&k_full[st]);
            if (i + 1 < n_tiles) {
                find(i + 1);
                tc_load<TYPE, D>(k, p.kv.k, p.kv.k_scale, row, x);
            }
            if (!__all_sync(0xffffffffu, wait_or_abort<20>(&v_free[st], ph ^ 1u, &s_abort, p.err))) break;
#pragma unroll
            for (int n = 0; n < S::NL; ++n) {
                const float f = tc_store<TYPE, D, true>(v, n, sv + st * S::KV_BYTES, n * S::ROWS + r0, x, there >> n & 1, masked);
                if (x == 0) v_scale[st][n * S::ROWS + r0] = there >> n & 1 ? f : 0.0f;
            }
            fence_async_smem();
            mbar_arrive(&v_full[st]);
            if (i + 1 < n_tiles) tc_load<TYPE, D>(v, p.kv.v, p.kv.v_scale, row, x);
        }
    } else if (lane == 0) {
        // ------------------------------------------------------------ products
        constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t) (KT >> 3) << 17) | ((128u >> 4) << 24);
        constexpr uint32_t IDESC_O = (1u << 4) | (1u << 16) | ((uint32_t) (D >> 3) << 17) | ((128u >> 4) << 24);    // second operand: head_dim contiguous
        auto values = [&](int i) {
            const int st = i & 1;
            const uint32_t ph = (i >> 1) & 1;
            if (!wait_or_abort(&p_full[st], ph, &s_abort, p.err) || !wait_or_abort(&v_full[st], ph, &s_abort, p.err)) return false;
            tc_fence_after();
            const uint32_t b = smem_u32(sv + st * S::KV_BYTES);
#pragma unroll
            for (int k = 0; k < KT / 16; ++k)
                umma_f16_ts(tmem + S::T_O, tmem + S::T_P + st * (KT / 2) + 8 * k, umma_desc_v(b + 2048 * k, KT * 128), IDESC_O, i > 0 || k > 0);
            umma_commit(&v_free[st]);
            umma_commit(&pv_done[st]);
            return true;
        };
        bool ok = true;
        for (int i = 0; i < n_tiles && ok; ++i) {
            const int st = i & 1;
            const uint32_t ph = (i >> 1) & 1;
            ok = wait_or_abort(&k_full[st], ph, &s_abort, p.err) && wait_or_abort(&s_free[st], ph ^ 1u, &s_abort, p.err);
            if (!ok) break;
            tc_fence_after();
            const uint32_t a = smem_u32(sq), b = smem_u32(sk + st * S::KV_BYTES);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                umma_f16(tmem + S::T_S + st * KT, umma_desc_k128(a + (k / 4) * (TC_ROWS * 128) + (k % 4) * 32),
                         umma_desc_k128(b + (k / 4) * (KT * 128) + (k % 4) * 32), IDESC_S, k > 0);
            umma_commit(&s_full[st]);
            umma_commit(&k_free[st]);
            if (i > 0) ok = values(i - 1);
        }
        if (ok && n_tiles) values(n_tiles - 1);
    }

    // ---- teardown: every wait above is bounded; the softmax warps have waited for the last product
    if (s_abort) {
        // products that were issued but not waited for end within microseconds: a bounded grace period
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) { }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == TC_SOFTMAX_WARPS + TC_PRODUCER_WARPS) tmem_dealloc(tmem, 512);
}

}  // namespace b200moe
