/* Causal attention over packed prompts (include/glint_serve.h).
 *
 * k_attend_prompt — a workgroup of 4 waves takes 128 query rows of one head, 32 a wave, and
 *   walks the keys in tiles of 64 through LDS. Scores are formed transposed,
 *   S^T = K Q^T on the 32x32x16 bf16 matrix instruction, so that a lane holds 32 keys of one
 *   query row: maximum and sum are in-lane but for one exchange of the wave's halves, and the
 *   weights feed O^T = V^T P^T as they lie (the order of the keys inside a product is free).
 *   V^T operands come from the row-major V tile by the transposing LDS read. */
#include "glint_common.h"
#include "glint_serve.h"

typedef __bf16 ap_bf16x8 __attribute__((ext_vector_type(8)));
typedef float ap_f32x16 __attribute__((ext_vector_type(16)));
typedef short ap_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ap_s16x4 ap_lds_s16x4;

#define AP_WAVES 4
#define AP_T (64 * AP_WAVES)
#define AP_ROWS (32 * AP_WAVES)
#define AP_KEYS 64

union ApFrag {
    uint32_t u[4];
    glint_u32x4 v;
    ap_s16x4 h[2];
    ap_bf16x8 f;
};

struct ApArgs {
    const uint16_t *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    const int32_t *cu_q, *cu_k;
    int64_t Tq, Tk;
    int max_q, Hq, G;
    float scale2; /* scale * log2 e */
    uint16_t *out;
};

template <int D>
__global__ __launch_bounds__(AP_T) void k_attend_prompt(ApArgs A) {
    constexpr int CH = D / 8; /* 16-B chunks of a row */
    __shared__ __attribute__((aligned(16))) uint16_t kt[AP_KEYS * D], vt[AP_KEYS * D];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 31, half = lane >> 5;
    const int hq = blockIdx.y, h = hq / A.G, b = blockIdx.z;
    const int64_t q0 = A.cu_q[b], k0 = A.cu_k[b];
    const int64_t q1 = A.cu_q[b + 1], k1 = A.cu_k[b + 1];
    if (q0 < 0 || q1 <= q0 || q1 > A.Tq)
        return;
    const int nq = (int)min(q1 - q0, (int64_t)A.max_q);
    const int nk = k0 >= 0 && k1 > k0 && k1 <= A.Tk ? (int)(k1 - k0) : 0;
    const int r0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * AP_ROWS; /* the longest rows first */
    if (r0 >= nq)
        return;
    const int row = r0 + 32 * wave + col;
    const int64_t gap = nk - (q1 - q0); /* row i's last key is i + gap */
    const int last = row < nq ? (int)max((int64_t)-1, row + gap) : -1;

    ApFrag qf[D / 16];
    {
        const uint16_t *qr = A.q + (q0 + min(row, nq - 1)) * A.q_st + hq * A.q_sh;
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
            qf[s].v = *(const glint_u32x4 *)(qr + 16 * s + 8 * half);
    }
    ap_f32x16 o[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            o[d][i] = 0.f;
    float m = -INFINITY, l = 0.f;

    const int64_t far = min(r0 + AP_ROWS, nq) - 1 + gap; /* the last key of the last row */
    const int ntiles = far < 0 ? 0 : (int)(far / AP_KEYS) + 1;
    const uint16_t *kb = A.k + k0 * A.k_st + h * A.k_sh, *vb = A.v + k0 * A.v_st + h * A.v_sh;
    for (int t = 0; t < ntiles; ++t) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < AP_KEYS * CH / AP_T; ++i) {
            const int u = threadIdx.x + i * AP_T, r = u / CH, c = u % CH;
            const int key = t * AP_KEYS + r;
            glint_u32x4 kv = {0, 0, 0, 0}, vv = {0, 0, 0, 0};
            if (key < nk) {
                kv = *(const glint_u32x4 *)(kb + key * A.k_st + 8 * c);
                vv = *(const glint_u32x4 *)(vb + key * A.v_st + 8 * c);
            }
            *(glint_u32x4 *)(kt + r * D + 8 * (c ^ (r & 7))) = kv;
            *(glint_u32x4 *)(vt + r * D + 8 * c) = vv;
        }
        __syncthreads();
        ap_f32x16 sc[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                sc[a][i] = 0.f;
            const int r = 32 * a + col;
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
                ApFrag f;
                f.v = *(const glint_u32x4 *)(kt + r * D + 8 * ((2 * s + half) ^ (r & 7)));
                sc[a] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.f, qf[s].f, sc[a], 0, 0, 0);
            }
        }
        /* element i of tile a is key 32 a + 8 (i / 4) + 4 half + i % 4 */
        const int first = t * AP_KEYS + 4 * half;
        float top = -INFINITY;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = first + 32 * a + 8 * (i >> 2) + (i & 3);
                const float x = key <= last ? sc[a][i] * A.scale2 : -INFINITY;
                sc[a][i] = x;
                top = fmaxf(top, x);
            }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.f : mn;
        const float keep = __builtin_amdgcn_exp2f(m - base);
        m = mn;
        float sum = 0.f, high = 0.f;
        ApFrag pf[4], rest[4];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(sc[a][i] - base);
                sum += p;
                high = fmaxf(high, p);
                pf[2 * a + (i >> 3)].f[i & 7] = (__bf16)p;
                sc[a][i] = p;
            }
        l = fmaf(l, keep, sum);
        /* A weight's bf16 rounding (2^-8) averages out over many keys and does not where few hold
         * the sum: a tile with a weight above 1 / 16 of some row's sum so far is multiplied by
         * what the rounding left as well. */
        const bool few = __any(high * 16.f > l + __shfl_xor(l, 32, 64));
        if (few) {
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    rest[2 * a + (i >> 3)].f[i & 7] = (__bf16)(sc[a][i] - (float)pf[2 * a + (i >> 3)].f[i & 7]);
        }
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                o[d][i] *= keep;
        /* step s multiplies keys 16 s + 8 j / 4 ... as the weights lie: keys 16 s + 4 half +
         * 0..3, then 8 on. A 16-lane group reads 4 keys x 16 dimensions: lane i addresses key
         * i / 4, dimensions 4 (i % 4), and receives dimension i of the 4 keys. */
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                ApFrag f;
                const int key = 16 * s + 4 * half + ((lane & 15) >> 2);
                const int dim = 32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ap_lds_s16x4 *)(vt + key * D + dim));
                f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ap_lds_s16x4 *)(vt + (key + 8) * D + dim));
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.f, pf[s].f, o[d], 0, 0, 0);
                if (few)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.f, rest[s].f, o[d], 0, 0, 0);
            }
    }
    l += __shfl_xor(l, 32, 64);
    if (row >= nq)
        return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t *dst = A.out + ((q0 + row) * A.Hq + hq) * D;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            glint_u32x2 two;
            two.x = glint_f32_to_bf16(o[d][i] * inv) | (uint32_t)glint_f32_to_bf16(o[d][i + 1] * inv) << 16;
            two.y = glint_f32_to_bf16(o[d][i + 2] * inv) | (uint32_t)glint_f32_to_bf16(o[d][i + 3] * inv) << 16;
            *(glint_u32x2 *)(dst + 32 * d + 2 * i + 4 * half) = two;
        }
}

GLINT_API int glint_attend_prompt(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, const uint16_t *k,
                                  int64_t k_stride_t, int64_t k_stride_h, const uint16_t *v, int64_t v_stride_t,
                                  int64_t v_stride_h, const int32_t *cu_q, const int32_t *cu_k, int64_t Tq, int64_t Tk,
                                  int B, int max_q, int Hq, int H, int D, float scale, uint16_t *out,
                                  struct ihipStream_t *stream) {
    if (!q || !k || !v || !cu_q || !cu_k || !out)
        return -1;
    if (B < 0 || B > 65535 || max_q < 0 || max_q > (1 << 30) || H < 1 || Hq < H || Hq > 65535 || Hq % H ||
        (D != 64 && D != 128) || Tq < 0 || Tk < 0)
        return -2;
    if (!glint_aligned(q, 16) || !glint_aligned(k, 16) || !glint_aligned(v, 16) || !glint_aligned(out, 8) ||
        ((q_stride_t | q_stride_h | k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7))
        return -2;
    if (B == 0 || Tq == 0 || max_q == 0)
        return 0;
    const ApArgs a{q, k, v, q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h, cu_q, cu_k, Tq, Tk,
                   max_q, Hq, Hq / H, scale * 1.44269504088896341f, out};
    const dim3 grid((unsigned)((max_q + AP_ROWS - 1) / AP_ROWS), Hq, B);
    if (D == 64)
        k_attend_prompt<64><<<grid, AP_T, 0, stream>>>(a);
    else
        k_attend_prompt<128><<<grid, AP_T, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
