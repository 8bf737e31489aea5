/* The 4-bit key/value cache: append and gather (include/glint_serve.h).
 *
 * Both move bytes: a token and head of D dimensions is 4 D bytes in BF16 (8 D in FP32) on one side and
 * D + 8 D / 64 on the other. Calls of few tokens are a launch and one load's latency after another.
 *
 * k_kv4_append — a row of 16 lanes encodes one 64-block of one token's key or value, four
 *   elements a lane; 8 tokens of 8 heads in 3.5 us.
 * k_kv4_gather — a thread reads one byte of a key row (two adjacent dimensions) or of a value
 *   column (dimensions 16 apart) and writes its two BF16; 8 tokens in 2.8 us.
 * k_kv4_append_tile, k_kv4_gather_tile — 32 tokens of one head a workgroup, for prompts: without
 *   them a value's bytes are written and read one by one, 64 B apart. 4096 tokens of 8 heads of
 *   128: append 11.1 us (1.9 TB/s; 23 element-wise), gather 10.9 us (2.0 TB/s; 17). Each is a chain
 *   of loads, LDS and stores, so the waves that a CU holds count: tiles of 64 tokens, half as many
 *   workgroups, took 12.0 and 14.2. */
#include "kv4_tile.h"

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

/* ------------------------------------------------------------------ tiles (kv4_tile.h) */
template <class E, int D>
__global__ __launch_bounds__(KV4_T) void k_kv4_append_tile(const E *__restrict__ k, const E *__restrict__ v, int64_t k_st,
                                                           int64_t k_sh, int64_t v_st, int64_t v_sh,
                                                           const int64_t *__restrict__ slots, int64_t T, int H,
                                                           uint8_t *__restrict__ k_hole, float *__restrict__ k_absmax,
                                                           uint8_t *__restrict__ v_hole, float *__restrict__ v_absmax,
                                                           int64_t nslots) {
    constexpr int NB = D / 64, ROWS = KV4_T / 8, PASSES = KT_TOKENS * NB / ROWS;
    __shared__ Kv4Bucket buckets[KV4_BUCKETS];
    __shared__ int64_t place[KT_COLS];
    __shared__ __attribute__((aligned(16))) uint8_t vt[(D / 2) * KT_COLS];
    __shared__ float scale[2][NB][KT_COLS];
    const int64_t t0 = (int64_t)blockIdx.x * KT_TOKENS;
    const int h = blockIdx.y, e = threadIdx.x & 7, r = threadIdx.x >> 3;
    kv4_fill_buckets(buckets);
    const int shift = kt_slots(slots, t0, T, nslots, place);
    __syncthreads();
#pragma unroll
    for (int is_v = 0; is_v < 2; ++is_v) {
        float w[PASSES][8];
#pragma unroll
        for (int i = 0; i < PASSES; ++i) { /* every load first */
            const int item = r + i * ROWS, j = item / NB, b = item % NB;
            const int64_t t = min(t0 + j, T - 1);
            kt_load8<D>((is_v ? v + t * v_st + h * v_sh : k + t * k_st + h * k_sh) + 64 * b + 8 * e, w[i]);
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int item = r + i * ROWS, j = item / NB, b = item % NB, c = j + shift;
            float s;
            const uint32_t code = kt_code8<sizeof(E) == 2>(buckets, w[i], s);
            const int64_t slot = place[c];
            if (e == 0)
                scale[is_v][b][c] = s;
            if (!is_v) {
                if (slot >= 0)
                    *(uint32_t *)(k_hole + (((slot >> 6) * H + h) * KV4_PAGE + (slot & 63)) * (D / 2) +
                                  kv4_k_byte<NB>(64 * b + 8 * e)) = code;
            } else {
                kt_put_value<KT_COLS>(vt + c, 64 * b, e, code);
            }
        }
    }
    __syncthreads();
    kt_store_values<D>(vt, place, h, H, v_hole);
    for (int u = threadIdx.x; u < 2 * NB * KT_COLS; u += KV4_T) {
        const int c = u % KT_COLS, b = u / KT_COLS % NB, is_v = u / (KT_COLS * NB);
        const int64_t p = place[c];
        if (p >= 0)
            (is_v ? v_absmax : k_absmax)[(((p >> 6) * H + h) * NB + b) * KV4_PAGE + (p & 63)] = scale[is_v][b][c];
    }
}

/* A thread writes 8 dimensions of a token: keys from their 4 bytes, values from LDS. */
template <int D>
__global__ __launch_bounds__(KV4_T) void k_kv4_gather_tile(const int64_t *__restrict__ slots, int64_t T, int H,
                                                           const uint8_t *__restrict__ k_hole,
                                                           const float *__restrict__ k_absmax,
                                                           const uint8_t *__restrict__ v_hole,
                                                           const float *__restrict__ v_absmax, int64_t nslots,
                                                           uint16_t *__restrict__ k, uint16_t *__restrict__ v) {
    constexpr int NB = D / 64, CH = D / 8;
    __shared__ int64_t place[KT_COLS];
    __shared__ __attribute__((aligned(16))) uint8_t vt[(D / 2) * KT_COLS];
    __shared__ float par[16 * 32]; /* 32 copies, one a bank */
    const int64_t t0 = (int64_t)blockIdx.x * KT_TOKENS;
    const int h = blockIdx.y;
    for (int i = threadIdx.x; i < 16 * 32; i += KV4_T)
        par[i] = kKv4Parent[i >> 5];
    const int shift = kt_slots(slots, t0, T, nslots, place);
    __syncthreads();
    const float *mine = par + (threadIdx.x & 31);
    for (int u = threadIdx.x; u < (D / 2) * KT_GROUPS; u += KV4_T) {
        const int row = u / KT_GROUPS, c = 4 * (u % KT_GROUPS);
        uint32_t word = 0;
        const int64_t s = kt_word(place, c);
        if (s >= 0) {
            word = *(const uint32_t *)(v_hole + (((s >> 6) * H + h) * (D / 2) + row) * KV4_PAGE + (s & 63));
        } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int64_t p = place[c + x];
                if (p >= 0)
                    word |= (uint32_t)v_hole[(((p >> 6) * H + h) * (D / 2) + row) * KV4_PAGE + (p & 63)] << (8 * x);
            }
        }
        *(uint32_t *)(vt + row * KT_COLS + c) = word;
    }
    __syncthreads();
#pragma unroll 4
    for (int u = threadIdx.x; u < KT_TOKENS * CH; u += KV4_T) {
        const int j = u / CH, d = 8 * (u % CH), c = j + shift, b = d >> 6;
        const int64_t t = t0 + j, p = place[c];
        if (t >= T)
            break;
        const int64_t ph = max(p, (int64_t)0) / KV4_PAGE * H + h;
        const int at = (int)(max(p, (int64_t)0) & 63);
        const uint32_t kw = *(const uint32_t *)(k_hole + (ph * KV4_PAGE + at) * (D / 2) + kv4_k_byte<NB>(d));
        const float ks = k_absmax[(ph * NB + b) * KV4_PAGE + at], vs = v_absmax[(ph * NB + b) * KV4_PAGE + at];
        const uint8_t *vr = vt + kv4_v_row(d) * KT_COLS + c;
        const int up = d & 16 ? 4 : 0;
        glint_u32x4 ko = {0, 0, 0, 0}, vo = {0, 0, 0, 0};
        if (p >= 0) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                ko[x] = glint_cvt_bf16x2(mine[((kw >> (8 * x)) & 15u) * 32] * ks, mine[((kw >> (8 * x + 4)) & 15u) * 32] * ks);
                const uint32_t a = (uint32_t)vr[2 * x * KT_COLS] >> up, z = (uint32_t)vr[(2 * x + 1) * KT_COLS] >> up;
                vo[x] = glint_cvt_bf16x2(mine[(a & 15u) * 32] * vs, mine[(z & 15u) * 32] * vs);
            }
        }
        *(glint_u32x4 *)(k + (t * H + h) * D + d) = ko;
        *(glint_u32x4 *)(v + (t * H + h) * D + d) = vo;
    }
}

/* When tiles are taken. A workgroup of them runs 5 to 7 us however little it has, so they want most of
 * the device's workgroups, and half their tokens. us, BF16, 128 dimensions, element-wise against tiles:
 *   tokens x heads   700 x 8      850 x 8      1250 x 8     1536 x 8     2048 x 8      4096 x 8
 *   append           6.7, 7.0     7.4, 7.0     9.8, 7.5     11.0, 7.7    13.7, 8.1     23.3, 11.1
 *   gather           5.4, 7.5     5.9, 7.3     7.4, 8.2     8.4, 7.5     10.5, 7.8     17.4, 10.9
 *   tokens x heads   16 x 512     16 x 1024
 *   append           7.8, 7.5     12.6, 9.9 */
#define KV4_TILE_APPEND 6144 /* tokens of one head */
#define KV4_TILE_GATHER 10240
#define KV4_TILE_T 16
static bool kv4_tiles(int64_t T, int H, int64_t from) { return T >= KV4_TILE_T && T * H >= from; }

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
static void kv4_append_tiles(const void *k, const void *v, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
                             const int64_t *slots, int64_t T, int H, int D, uint8_t *k_hole, float *k_absmax,
                             uint8_t *v_hole, float *v_absmax, int64_t pages, hipStream_t stream) {
    const dim3 g((unsigned)((T + KT_TOKENS - 1) / KT_TOKENS), H);
    if (D == 64)
        k_kv4_append_tile<E, 64><<<g, KV4_T, 0, stream>>>((const E *)k, (const E *)v, k_st, k_sh, v_st, v_sh, slots, T, H,
                                                          k_hole, k_absmax, v_hole, v_absmax, pages * 64);
    else
        k_kv4_append_tile<E, 128><<<g, KV4_T, 0, stream>>>((const E *)k, (const E *)v, k_st, k_sh, v_st, v_sh, slots, T, H,
                                                           k_hole, k_absmax, v_hole, v_absmax, pages * 64);
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
    /* the tiles load 8 elements at once */
    const bool tiles = kv4_tiles(T, H, KV4_TILE_APPEND) && glint_aligned(k, 16) && glint_aligned(v, 16) &&
                       !((k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7);
    if (tiles && elt == GLINT_KV_BF16)
        kv4_append_tiles<uint16_t>(k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, slots, T, H, D, k_hole, k_absmax,
                                   v_hole, v_absmax, pages, stream);
    else if (tiles)
        kv4_append_tiles<float>(k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, slots, T, H, D, k_hole, k_absmax,
                                v_hole, v_absmax, pages, stream);
    else if (elt == GLINT_KV_BF16)
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
    const dim3 tiles((unsigned)((T + KT_TOKENS - 1) / KT_TOKENS), H);
    if (kv4_tiles(T, H, KV4_TILE_GATHER) && glint_aligned(k, 16) && glint_aligned(v, 16)) {
        if (D == 64)
            k_kv4_gather_tile<64><<<tiles, KV4_T, 0, stream>>>(slots, T, H, k_hole, k_absmax, v_hole, v_absmax, pages * 64, k, v);
        else
            k_kv4_gather_tile<128><<<tiles, KV4_T, 0, stream>>>(slots, T, H, k_hole, k_absmax, v_hole, v_absmax, pages * 64, k, v);
    } else if (D == 64)
        k_kv4_gather<64><<<dim3(g, 2), KV4_T, 0, stream>>>(slots, T, H, k_hole, k_absmax, v_hole, v_absmax, pages * 64,
                                                           k, v);
    else
        k_kv4_gather<128><<<dim3(g, 2), KV4_T, 0, stream>>>(slots, T, H, k_hole, k_absmax, v_hole, v_absmax, pages * 64,
                                                            k, v);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
