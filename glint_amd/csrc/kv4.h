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

/* Byte of dimension pair (d, d + 1), d even, in a key row of NB blocks. */
template <int NB>
__host__ __device__ __forceinline__ int kv4_k_byte(int d) {
    return (((d & 63) >> 4) * NB + (d >> 6)) * 8 + ((d & 15) >> 1);
}
/* Row of dimension d in a value page; bit 4 of d says which nibble. */
__host__ __device__ __forceinline__ int kv4_v_row(int d) { return ((d >> 5) << 4) + (d & 15); }

#endif
