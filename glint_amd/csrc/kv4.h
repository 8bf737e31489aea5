/* The 4-bit key/value cache's layout and code rule (include/glint_serve.h). */
#ifndef GLINT_KV4_H_
#define GLINT_KV4_H_

#include "glint_common.h"
#include "glint_serve.h"

#define KV4_PAGE GLINT_KV_PAGE

static __constant__ float kKv4Parent[16] = GLINT_PARENT_INIT;

/* The hole of v is the number of these that lie below it: KV4_EDGES[k] is the largest float
 * whose first minimum of |v - PARENT| is at most k. */
#define KV4_EDGES                                                                                                      \
    {-0x1.b239b2p-1f, -0x1.38a4e2p-1f, -0x1.d709p-2f, -0x1.5bd4eep-2f, -0x1.e079dap-3f, -0x1.1a7178p-3f,              \
     -0x1.74f0e2p-5f, 0x1.45f5fep-5f, 0x1.ec90c4p-4f, 0x1.a0cfcp-3f, 0x1.2b05a8p-2f, 0x1.8ea7f2p-2f, 0x1.00da06p-1f,  \
     0x1.491b5ep-1f, 0x1.b913b2p-1f}

__device__ __forceinline__ uint32_t kv4_code(float v) {
    constexpr float edge[15] = KV4_EDGES;
    uint32_t c = 0;
#pragma unroll
    for (int k = 0; k < 15; ++k)
        c += v > edge[k] ? 1u : 0u; /* NaN: 0 */
    return c;
}

/* The same by a table of buckets a sixteenth wide, of which each holds one edge at most (they lie
 * 0.08 apart): hole = base + (v > edge). fmaf(v, 16, 2^23 + 16) is an integer in [2^23, 2^23 + 32]
 * for v in [-1, 1]. */
#define KV4_BUCKETS 33
#define KV4_MAGIC 8388624.f       /* 2^23 + 16 */
#define KV4_MAGIC_BITS 0x4B000000u /* 2^23 */
struct Kv4Bucket {
    float edge;
    uint32_t base;
};
__device__ __forceinline__ void kv4_fill_buckets(Kv4Bucket *t) { /* a barrier follows */
    constexpr float edge[15] = KV4_EDGES;
    const int i = threadIdx.x;
    if (i < KV4_BUCKETS) {
        /* values that round to the bucket's integer: half a bucket on either side */
        const float low = (i - 16 - 0.5f) * 0.0625f;
        uint32_t base = 0;
        float e = INFINITY;
#pragma unroll
        for (int k = 14; k >= 0; --k) {
            if (edge[k] >= low)
                e = edge[k];
            else
                ++base;
        }
        t[i] = Kv4Bucket{e, base};
    }
}
__device__ __forceinline__ uint32_t kv4_code(const Kv4Bucket *t, float v) { /* |v| <= 1, or NaN: 0 */
    const Kv4Bucket e = t[__float_as_uint(fmaf(fmaxf(v, -1.f), 16.f, KV4_MAGIC)) - KV4_MAGIC_BITS];
    return e.base + (v > e.edge ? 1u : 0u);
}

/* The attention kernels' table holds PARENT * KV4_ALPHA, whose f16 roundings are smaller and cancel: over the code
 * frequencies of normal values under a block-64 absmax (sigma 0.25 to 0.6 of it) and of even
 * ones, the mean error is at most 1.8e-6 of the absmax and the rms 3.9e-5, where PARENT's own
 * are 1.6e-5 and 9.5e-5. The mean counts: it is all that is left of the values' rounding in
 * the output of a long row, and at 8192 tokens of equal weight it alone was 0.8 of the bf16
 * output's rounding. */
#define KV4_ALPHA 1.458935f

/* Byte of dimension pair (d, d + 1), d even, in a key row of NB blocks. */
template <int NB>
__host__ __device__ __forceinline__ int kv4_k_byte(int d) {
    return (((d & 63) >> 4) * NB + (d >> 6)) * 8 + ((d & 15) >> 1);
}
/* Row of dimension d in a value page; bit 4 of d says which nibble. */
__host__ __device__ __forceinline__ int kv4_v_row(int d) { return ((d >> 5) << 4) + (d & 15); }

#endif
