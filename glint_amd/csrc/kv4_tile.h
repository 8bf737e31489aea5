/* Encoding rows of 8 dimensions a lane, and tiles of 32 tokens: what the kernels that fill the 4-bit cache share. */
#ifndef GLINT_KV4_TILE_H_
#define GLINT_KV4_TILE_H_

#include "kv4.h"

#define KV4_T 256

template <int CTRL>
__device__ __forceinline__ float kv4_max_dpp(float v) {
    return fmaxf(v, __int_as_float(glint_dpp<CTRL>(__float_as_int(v))));
}

/* A row of 8 lanes encodes a 64-block, 8 dimensions a lane: their quotients by one multiply where the
 * input is BF16 and the absmax ordinary (no code differs from the divide's, see
 * tests/native/check_encode_quotient.c), by the divide elsewhere. 8 nibbles, and the block's absmax. */
template <bool BF16>
__device__ __forceinline__ uint32_t kt_code8(const Kv4Bucket *buckets, const float (&w)[8], float &s) {
    s = 0.f; /* fmaxf leaves NaN out */
#pragma unroll
    for (int x = 0; x < 8; ++x)
        s = fmaxf(s, fabsf(w[x]));
    s = kv4_max_dpp<GLINT_DPP_QUAD_1032>(s);
    s = kv4_max_dpp<GLINT_DPP_QUAD_2301>(s);
    s = kv4_max_dpp<GLINT_DPP_ROW_HALF_MIRROR>(s);
    uint32_t code = 0;
    if (BF16 && s >= 0x1p-90f && s < 0x1p90f) {
        const float inv = 1.f / s;
#pragma unroll
        for (int x = 0; x < 8; ++x) /* NaN among them: an absmax that leaves it out is no bound for it */
            code |= kv4_code(buckets, w[x] * inv) << (4 * x);
    } else {
#pragma unroll
        for (int x = 0; x < 8; ++x)
            code |= kv4_code(buckets, s == 0.f ? 0.f : w[x] / s) << (4 * x);
    }
    return code;
}

/* The bytes of a value block's lane e (of the block at dimension d0) go to a column of rows STRIDE bytes
 * apart: dimensions 16 on are two lanes on, and this lane writes four of the pair's rows. */
template <int STRIDE>
__device__ __forceinline__ void kt_put_value(uint8_t *column, int d0, int e, uint32_t code) {
    const uint32_t other = (uint32_t)glint_dpp<GLINT_DPP_QUAD_2301>((int)code);
    const int up = e & 2 ? 16 : 0;
    const uint32_t lo = (e & 2 ? other : code) >> up, hi = (e & 2 ? code : other) >> up;
    uint8_t *row = column + (kv4_v_row(d0 + 8 * (e & ~2)) + (e & 2 ? 4 : 0)) * STRIDE;
#pragma unroll
    for (int x = 0; x < 4; ++x)
        row[x * STRIDE] = (uint8_t)(((lo >> (4 * x)) & 15u) | ((hi >> (4 * x)) & 15u) << 4);
}

/* 32 tokens of one head a workgroup. A value column lies a byte a token, 64 B apart, so values
 * pass through LDS: columns there are shifted by the first token's place modulo 4, so that four
 * tokens whose slots follow each other, as a prompt's do, are one aligned word on both sides;
 * other tokens go byte by byte. */
#define KT_TOKENS 32
#define KT_COLS (KT_TOKENS + 4) /* the shift */
#define KT_GROUPS (KT_COLS / 4)

/* The slots of a tile, by shifted column; -1 where there is no token. */
__device__ __forceinline__ int kt_slots(const int64_t *slots, int64_t t0, int64_t T, int64_t nslots, int64_t *place) {
    const int64_t first = slots[t0];
    const int shift = first >= 0 && first < nslots ? (int)(first & 3) : 0;
    for (int c = threadIdx.x; c < KT_COLS; c += KV4_T) {
        const int64_t t = t0 + c - shift;
        const int64_t s = c >= shift && c - shift < KT_TOKENS && t < T ? slots[t] : -1;
        place[c] = s < nslots ? s : -1;
    }
    return shift;
}
/* Whether columns c .. c + 3 are four slots in a row, the first a multiple of 4: its place, or -1. */
__device__ __forceinline__ int64_t kt_word(const int64_t *place, int c) {
    const int64_t s = place[c];
    return s >= 0 && (s & 3) == 0 && place[c + 1] == s + 1 && place[c + 2] == s + 2 && place[c + 3] == s + 3 ? s : -1;
}

template <int D>
__device__ __forceinline__ void kt_load8(const uint16_t *p, float (&w)[8]) {
    const glint_u32x4 u = *(const glint_u32x4 *)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[2 * i] = glint_bf16lo(u[i]);
        w[2 * i + 1] = glint_bf16hi(u[i]);
    }
}
template <int D>
__device__ __forceinline__ void kt_load8(const float *p, float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const glint_f32x4 u = ((const glint_f32x4 *)p)[i];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w[4 * i + k] = u[k];
    }
}

/* A tile's value columns from LDS to head h of the pages. */
template <int D>
__device__ __forceinline__ void kt_store_values(const uint8_t *vt, const int64_t *place, int h, int H, uint8_t *v_hole) {
    for (int u = threadIdx.x; u < (D / 2) * KT_GROUPS; u += KV4_T) {
        const int row = u / KT_GROUPS, c = 4 * (u % KT_GROUPS);
        const uint32_t word = *(const uint32_t *)(vt + row * KT_COLS + c);
        const int64_t s = kt_word(place, c);
        if (s >= 0) {
            *(uint32_t *)(v_hole + (((s >> 6) * H + h) * (D / 2) + row) * KV4_PAGE + (s & 63)) = word;
        } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int64_t p = place[c + x];
                if (p >= 0)
                    v_hole[(((p >> 6) * H + h) * (D / 2) + row) * KV4_PAGE + (p & 63)] = (uint8_t)(word >> (8 * x));
            }
        }
    }
}

#endif
