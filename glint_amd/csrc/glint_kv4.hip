/* The 4-bit key/value cache: append and gather (include/glint_serve.h).
 *
 * k_kv4_append — a row of 16 lanes encodes one 64-block of one token's key or value, four
 *   elements a lane.
 * k_kv4_gather — a thread reads one byte of a key row (two adjacent dimensions) or of a value
 *   column (dimensions 16 apart) and writes its two BF16. */
#include "kv4.h"

#define KV4_T 256

template <class E>
__device__ __forceinline__ void kv4_load4(const E *p, float (&w)[4]);
template <>
__device__ __forceinline__ void kv4_load4(const uint16_t *p, float (&w)[4]) {
    const uint2 u = *(const uint2 *)p;
    w[0] = glint_bf16lo(u.x);
    w[1] = glint_bf16hi(u.x);
    w[2] = glint_bf16lo(u.y);
    w[3] = glint_bf16hi(u.y);
}
template <>
__device__ __forceinline__ void kv4_load4(const float *p, float (&w)[4]) {
    const glint_f32x4 u = *(const glint_f32x4 *)p;
    w[0] = u.x;
    w[1] = u.y;
    w[2] = u.z;
    w[3] = u.w;
}

template <int CTRL>
__device__ __forceinline__ float kv4_max_dpp(float v) {
    return fmaxf(v, __int_as_float(glint_dpp<CTRL>(__float_as_int(v))));
}

template <class E, int D>
__global__ __launch_bounds__(KV4_T) void k_kv4_append(const E *__restrict__ k, const E *__restrict__ v,
                                                      int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
                                                      const int64_t *__restrict__ slots, int64_t T, int H,
                                                      uint8_t *__restrict__ k_hole, float *__restrict__ k_absmax,
                                                      uint8_t *__restrict__ v_hole, float *__restrict__ v_absmax,
                                                      int64_t nslots) {
    constexpr int NB = D / 64;
    const int64_t item = ((int64_t)blockIdx.x * KV4_T + threadIdx.x) >> 4;
    const int e = threadIdx.x & 15, b = (int)(item % NB);
    const int64_t th = item / NB, t = th / H;
    const int h = (int)(th % H);
    if (t >= T)
        return;
    const int64_t slot = slots[t];
    if (slot < 0 || slot >= nslots)
        return;
    const bool is_v = blockIdx.y != 0;
    float w[4];
    kv4_load4(is_v ? v + t * v_st + h * v_sh + 64 * b + 4 * e : k + t * k_st + h * k_sh + 64 * b + 4 * e, w);
    float s = 0.f; /* fmaxf leaves NaN out */
#pragma unroll
    for (int i = 0; i < 4; ++i)
        s = fmaxf(s, fabsf(w[i]));
    s = kv4_max_dpp<GLINT_DPP_QUAD_1032>(s);
    s = kv4_max_dpp<GLINT_DPP_QUAD_2301>(s);
    s = kv4_max_dpp<GLINT_DPP_ROW_HALF_MIRROR>(s);
    s = kv4_max_dpp<GLINT_DPP_ROW_MIRROR>(s);
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        c[i] = kv4_code(s == 0.f ? 0.f : w[i] / s);
    const int64_t ph = (slot >> 6) * H + h;
    const int at = (int)(slot & 63);
    if (!is_v) {
        const uint32_t two = c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12;
        *(uint16_t *)(k_hole + (ph * KV4_PAGE + at) * (D / 2) + kv4_k_byte<NB>(64 * b + 4 * e)) = (uint16_t)two;
        if (e == 0)
            k_absmax[(ph * NB + b) * KV4_PAGE + at] = s;
    } else {
        /* the other nibble's dimensions are 16 on: four lanes */
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = (uint32_t)__shfl_xor((int)c[i], 4, 64);
        uint8_t *row = v_hole + (ph * (D / 2) + kv4_v_row(64 * b + 4 * e)) * KV4_PAGE + at;
        if (e & 4) {
            row[2 * KV4_PAGE] = (uint8_t)(o[2] | c[2] << 4);
            row[3 * KV4_PAGE] = (uint8_t)(o[3] | c[3] << 4);
        } else {
            row[0] = (uint8_t)(c[0] | o[0] << 4);
            row[KV4_PAGE] = (uint8_t)(c[1] | o[1] << 4);
        }
        if (e == 0)
            v_absmax[(ph * NB + b) * KV4_PAGE + at] = s;
    }
}

template <int D>
__global__ __launch_bounds__(KV4_T) void k_kv4_gather(const int64_t *__restrict__ slots, int64_t T, int H,
                                                      const uint8_t *__restrict__ k_hole,
                                                      const float *__restrict__ k_absmax,
                                                      const uint8_t *__restrict__ v_hole,
                                                      const float *__restrict__ v_absmax, int64_t nslots,
                                                      uint16_t *__restrict__ k, uint16_t *__restrict__ v) {
    constexpr int NB = D / 64;
    __shared__ float par[16];
    if (threadIdx.x < 16)
        par[threadIdx.x] = kKv4Parent[threadIdx.x];
    __syncthreads();
    const int64_t item = (int64_t)blockIdx.x * KV4_T + threadIdx.x;
    const int64_t th = item / (D / 2), t = th / H;
    const int h = (int)(th % H), y = (int)(item % (D / 2));
    if (t >= T)
        return;
    const int64_t slot = slots[t];
    const bool held = slot >= 0 && slot < nslots;
    const int64_t ph = held ? (slot >> 6) * H + h : 0;
    const int at = held ? (int)(slot & 63) : 0;
    if (blockIdx.y == 0) {
        const int d = 2 * y;
        uint32_t two = 0;
        if (held) {
            const uint32_t c = k_hole[(ph * KV4_PAGE + at) * (D / 2) + kv4_k_byte<NB>(d)];
            const float s = k_absmax[(ph * NB + (d >> 6)) * KV4_PAGE + at];
            two = glint_f32_to_bf16(par[c & 15] * s) | (uint32_t)glint_f32_to_bf16(par[c >> 4] * s) << 16;
        }
        *(uint32_t *)(k + th * D + d) = two;
    } else {
        const int d = ((y >> 4) << 5) + (y & 15);
        uint16_t lo = 0, hi = 0;
        if (held) {
            const uint32_t c = v_hole[(ph * (D / 2) + y) * KV4_PAGE + at];
            const float s = v_absmax[(ph * NB + (d >> 6)) * KV4_PAGE + at];
            lo = glint_f32_to_bf16(par[c & 15] * s);
            hi = glint_f32_to_bf16(par[c >> 4] * s);
        }
        v[th * D + d] = lo;
        v[th * D + d + 16] = hi;
    }
}

/* Workgroups of KV4_T threads for n threads' work, or 0 where a grid cannot hold them. */
static unsigned kv4_grid(int64_t T, int64_t per_token) {
    if (T > ((int64_t)1 << 40) / per_token)
        return 0;
    const int64_t g = (T * per_token + KV4_T - 1) / KV4_T;
    return g < ((int64_t)1 << 31) / KV4_T ? (unsigned)g : 0;
}

static bool kv4_shape(int64_t T, int H, int D, int64_t pages) {
    return T >= 0 && H >= 1 && H <= 65535 && (D == 64 || D == 128) && pages >= 1 && pages < (int64_t)1 << 40;
}

template <class E>
static void kv4_append_launch(unsigned g, const void *k, const void *v, int64_t k_st, int64_t k_sh, int64_t v_st,
                              int64_t v_sh, const int64_t *slots, int64_t T, int H, int D, uint8_t *k_hole,
                              float *k_absmax, uint8_t *v_hole, float *v_absmax, int64_t pages, hipStream_t stream) {
    if (D == 64)
        k_kv4_append<E, 64><<<dim3(g, 2), KV4_T, 0, stream>>>((const E *)k, (const E *)v, k_st, k_sh, v_st, v_sh, slots,
                                                              T, H, k_hole, k_absmax, v_hole, v_absmax, pages * 64);
    else
        k_kv4_append<E, 128><<<dim3(g, 2), KV4_T, 0, stream>>>((const E *)k, (const E *)v, k_st, k_sh, v_st, v_sh, slots,
                                                               T, H, k_hole, k_absmax, v_hole, v_absmax, pages * 64);
}

GLINT_API int glint_kv4_append(const void *k, const void *v, int elt, int64_t k_stride_t, int64_t k_stride_h,
                               int64_t v_stride_t, int64_t v_stride_h, const int64_t *slots, int64_t T, int H, int D,
                               uint8_t *k_hole, float *k_absmax, uint8_t *v_hole, float *v_absmax, int64_t pages,
                               struct ihipStream_t *stream) {
    if (!k || !v || !slots || !k_hole || !k_absmax || !v_hole || !v_absmax)
        return -1;
    if (!kv4_shape(T, H, D, pages) || (elt != GLINT_KV_BF16 && elt != GLINT_KV_F32))
        return -2;
    const size_t al = elt == GLINT_KV_BF16 ? 8 : 16;
    if (!glint_aligned(k, al) || !glint_aligned(v, al) || !glint_aligned(k_hole, 16) || !glint_aligned(v_hole, 16) ||
        ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 3))
        return -2;
    if (T == 0)
        return 0;
    const unsigned g = kv4_grid(T, (int64_t)H * (D / 64) * 16);
    if (!g)
        return -2;
    if (elt == GLINT_KV_BF16)
        kv4_append_launch<uint16_t>(g, k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, slots, T, H, D, k_hole,
                                    k_absmax, v_hole, v_absmax, pages, stream);
    else
        kv4_append_launch<float>(g, k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, slots, T, H, D, k_hole,
                                 k_absmax, v_hole, v_absmax, pages, stream);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}

GLINT_API int glint_kv4_gather(const int64_t *slots, int64_t T, int H, int D, const uint8_t *k_hole,
                               const float *k_absmax, const uint8_t *v_hole, const float *v_absmax, int64_t pages,
                               uint16_t *k, uint16_t *v, struct ihipStream_t *stream) {
    if (!k || !v || !slots || !k_hole || !k_absmax || !v_hole || !v_absmax)
        return -1;
    if (!kv4_shape(T, H, D, pages) || !glint_aligned(k, 4) || !glint_aligned(v, 4))
        return -2;
    if (T == 0)
        return 0;
    const unsigned g = kv4_grid(T, (int64_t)H * (D / 2));
    if (!g)
        return -2;
    if (D == 64)
        k_kv4_gather<64><<<dim3(g, 2), KV4_T, 0, stream>>>(slots, T, H, k_hole, k_absmax, v_hole, v_absmax, pages * 64,
                                                           k, v);
    else
        k_kv4_gather<128><<<dim3(g, 2), KV4_T, 0, stream>>>(slots, T, H, k_hole, k_absmax, v_hole, v_absmax, pages * 64,
                                                            k, v);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
