/* Queries and keys normed per head and turned to their positions, and the same on the way into the 4-bit
 * cache (include/glint_serve.h).
 *
 * k_rotate — a workgroup takes rows (a token's heads, queries first) of one token: its rot / 2 angles are
 *   formed once, one a thread, and shared through LDS; then LPR lanes take a row, 8 dimensions each, and
 *   exchange the sum of its squares and what is paired across lanes. Angles, sines and cosines are formed in 64 bits, right at any position.
 *
 *   k_rotate of the cache's form encodes a key after its rounding, as kv4_append would encode what rotate_qk
 *   returns, in the lanes that hold it. Values of few tokens are further rows; of many, tiles of 32 tokens
 *   through LDS, as glint_kv4.hip's, workgroups of the same launch.
 *
 *   What bounds it: bytes, each read and written once, or the launch. 4095 tokens of 32 and 8 heads of 128: 84 MB
 *   in 15.8 us from Python (17.0 traced), 5.3 TB/s, the rate of a copy, of f32 rows 168 MB in 29 to 31; with another lane's dimensions
 *   read from memory again instead of exchanged 18.0. 4096 tokens into the cache 27 us for 88 MB, 3.3 TB/s: 1.27e7 vector
 *   instructions, 21 us of 1024 SIMDs at 4 clocks each and 2.4 GHz. 8 tokens: the kernel 4 us, a call from Python 14. */
#include <algorithm>

#include "kv4_tile.h"

#define KR_T 256

struct RotateArgs {
    const void *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    const int64_t *pos;
    const double *freqs;
    int64_t T;
    int Hq, H, D, rot, interleaved;
    double magnitude;
    float eps, inv_d;
    const void *q_norm, *k_norm;
    int norm_f32;
    void *q_out, *k_out;
    /* the cache's form */
    const int64_t *slots;
    uint8_t *k_hole, *v_hole;
    float *k_absmax, *v_absmax;
    int64_t nslots;
    int value_rows;  /* of a token among its rows: H, or 0 where tiles take them */
    unsigned tiles;  /* value tiles, the launch's last workgroups */
    int tile_blocks; /* of 32 tokens */
    int parts;       /* workgroups of a token */
};

/* cos and sin of an angle, in f64 up to the rounding at the end: a key's code may hinge on its last bit, and then
 * does not on how the angle was formed. |angle| < 2^51. */
__device__ __forceinline__ glint_f32x2 kr_turn(double angle, double magnitude) {
    const double magic = 0x1.8p52;
    const double shifted = fma(angle, 0x1.45f306dc9c883p-1, magic); /* its low bits are the nearest number of quarter turns */
    const int quarter = (int)__double_as_longlong(shifted) & 3;
    const double n = shifted - magic;
    double x = fma(n, -0x1.921fb54442d18p0, angle); /* pi / 2 in two parts */
    x = fma(n, -0x1.1a62633145c07p-54, x);          /* |x| <= pi / 4 */
    const double z = x * x;
    /* Taylor's sums; what they leave out: x^15 / 15! < 2^-45, x^16 / 16! < 2^-49 */
    double s = fma(z, 0x1.6124613a86d09p-33, -0x1.ae64567f544e4p-26);
    s = fma(z, s, 0x1.71de3a556c734p-19);
    s = fma(z, s, -0x1.a01a01a01a01ap-13);
    s = fma(z, s, 0x1.1111111111111p-7);
    s = fma(z, s, -0x1.5555555555555p-3);
    s = fma(x * z, s, x);
    double c = fma(z, -0x1.93974a8c07c9dp-37, 0x1.1eed8eff8d898p-29);
    c = fma(z, c, -0x1.27e4fb7789f5cp-22);
    c = fma(z, c, 0x1.a01a01a01a01ap-16);
    c = fma(z, c, -0x1.6c16c16c16c17p-10);
    c = fma(z, c, 0x1.5555555555555p-5);
    c = fma(z, c, -0.5);
    c = fma(z, c, 1.0);
    const float a = (float)((quarter & 1 ? s : c) * magnitude), b = (float)((quarter & 1 ? c : s) * magnitude);
    return glint_f32x2{(quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b};
}

/* 1 / sqrt(x) rounded once: a step of Newton's behind the instruction, which is off by a bit in one value of ten. What
 * x r r leaves of 1 is formed from exact products, good to 2^-47. */
__device__ __forceinline__ float kr_rsqrt(float x) {
    const float r = rsqrtf(x), h = x * r, l = fmaf(x, r, -h);
    const float y = fmaf(0.5f * r, fmaf(-l, r, fmaf(-h, r, 1.f)), r);
    return r > 0.f && r < INFINITY ? y : r; /* of 0 and of infinity as they are */
}

__device__ __forceinline__ void kr_store8(uint16_t *p, const float (&w)[8]) {
    glint_u32x4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        u[i] = glint_cvt_bf16x2(w[2 * i], w[2 * i + 1]);
    *(glint_u32x4 *)p = u;
}
__device__ __forceinline__ void kr_store8(float *p, const float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        ((glint_f32x4 *)p)[i] = glint_f32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
}
/* A norm's 8 weights from dimension d on; ones where there is no norm. */
__device__ __forceinline__ void kr_norm8(const void *norm, int f32, int d, float (&g)[8]) {
    if (!norm) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            g[i] = 1.f;
    } else if (f32) {
        kt_load8<0>((const float *)norm + d, g);
    } else {
        kt_load8<0>((const uint16_t *)norm + d, g);
    }
}

/* 32 tokens' values of one head into the cache. */
template <class E, int D>
__device__ __forceinline__ void kr_value_tile(const RotateArgs &A, const Kv4Bucket *buckets, int64_t *place, uint8_t *vt,
                                              float *scale) {
    constexpr int NB = D / 64, ROWS = KR_T / 8, PASSES = KT_TOKENS * NB / ROWS;
    const unsigned at = blockIdx.x - (gridDim.x - A.tiles);
    const int64_t t0 = (int64_t)(at % A.tile_blocks) * KT_TOKENS;
    const int h = at / A.tile_blocks, e = threadIdx.x & 7, r = threadIdx.x >> 3;
    float w[PASSES][8];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) { /* every load first */
        const int item = r + i * ROWS;
        kt_load8<D>((const E *)A.v + min(t0 + item / NB, A.T - 1) * A.v_st + h * A.v_sh + 64 * (item % NB) + 8 * e, w[i]);
    }
    const int shift = kt_slots(A.slots, t0, A.T, A.nslots, place);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int item = r + i * ROWS, b = item % NB, c = item / NB + shift;
        float s;
        const uint32_t code = kt_code8<sizeof(E) == 2>(buckets, w[i], s);
        if (e == 0)
            scale[b * KT_COLS + c] = s;
        kt_put_value<KT_COLS>(vt + c, 64 * b, e, code);
    }
    __syncthreads();
    kt_store_values<D>(vt, place, h, A.H, A.v_hole);
    for (int u = threadIdx.x; u < NB * KT_COLS; u += KR_T) {
        const int64_t p = place[u % KT_COLS];
        if (p >= 0)
            A.v_absmax[(((p >> 6) * A.H + h) * NB + u / KT_COLS) * KV4_PAGE + (p & 63)] = scale[u];
    }
}

/* E: the rows' type. LPR: lanes of a row, a power of two of D / 8 at least. CACHE: keys and values go into
 * the cache; D is then 8 LPR. */
template <class E, int LPR, bool CACHE>
__global__ __launch_bounds__(KR_T) void k_rotate(RotateArgs A) {
    constexpr int ROWS = KR_T / LPR; /* a pass */
    constexpr int CD = 8 * LPR;      /* D where CACHE */
    constexpr int NB = CD / 64;
    __shared__ __attribute__((aligned(16))) glint_f32x2 turn[128];
    __shared__ Kv4Bucket buckets[CACHE ? KV4_BUCKETS : 1];
    __shared__ int64_t place[CACHE ? KT_COLS : 1];
    __shared__ __attribute__((aligned(16))) uint8_t vt[CACHE ? (CD / 2) * KT_COLS : 1];
    __shared__ float scale[CACHE ? (NB + 1) * KT_COLS : 1];
    if constexpr (CACHE) {
        kv4_fill_buckets(buckets);
        if (blockIdx.x >= gridDim.x - A.tiles) {
            kr_value_tile<E, CD>(A, buckets, place, vt, scale);
            return;
        }
    }
    int64_t t = (int64_t)blockIdx.x / A.parts;
    const int part = (int)(blockIdx.x % A.parts);
    if (A.parts == 1) { /* neighbours' places in the cache share lines: neighbours go to one XCD, the workgroup's index modulo 8 */
        const int64_t per = A.T >> 3;
        t = t < 8 * per ? (t & 7) * per + (t >> 3) : t;
    }
    const int half = A.rot / 2, rows = A.Hq + A.H + (CACHE ? A.value_rows : 0);
    const double p = (double)A.pos[t];
    if ((int)threadIdx.x < half)
        turn[threadIdx.x] = kr_turn(p * A.freqs[threadIdx.x], A.magnitude);
    int64_t slot = -1;
    if constexpr (CACHE) {
        slot = A.slots[t];
        slot = slot < A.nslots ? slot : -1;
    }
    __syncthreads();
    const int c = threadIdx.x % LPR, d = 8 * c;
    const bool in = d < A.D, turned = d < A.rot;
    /* y_i = w_i cs_i + p_i sn_i, p_i the dimension that i is paired with, in lane `other` of the row */
    float cs[8], sn[8], gq[8], gk[8];
    kr_norm8(A.q_norm, A.norm_f32, in ? d : 0, gq);
    kr_norm8(A.k_norm, A.norm_f32, in ? d : 0, gk);
    int other = threadIdx.x & 63;
    if (!turned) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            cs[i] = 1.f;
            sn[i] = 0.f;
        }
    } else if (A.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const glint_f32x2 x = turn[4 * c + i];
            cs[2 * i] = cs[2 * i + 1] = x.x;
            sn[2 * i] = -x.y;
            sn[2 * i + 1] = x.y;
        }
    } else {
        const bool first = d < half;
        other += first ? half / 8 : -half / 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const glint_f32x2 x = turn[(first ? d : d - half) + i];
            cs[i] = x.x;
            sn[i] = first ? -x.y : x.y;
        }
    }
    /* a wave ends with its own last row: 40 rows are 10 waves' */
    for (int row = part * ROWS + (int)threadIdx.x / LPR; row - (int)(threadIdx.x & 63) / LPR < rows; row += A.parts * ROWS) {
        const bool is_v = CACHE && row >= A.Hq + A.H, is_k = row >= A.Hq && !is_v, live = in && row < rows;
        const int h = is_v ? row - A.Hq - A.H : is_k ? row - A.Hq : row;
        const E *from = is_v   ? (const E *)A.v + t * A.v_st + h * A.v_sh
                        : is_k ? (const E *)A.k + t * A.k_st + h * A.k_sh
                               : (const E *)A.q + t * A.q_st + h * A.q_sh;
        float w[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i] = y[i] = 0.f;
        if (live)
            kt_load8<0>(from + d, w);
        if (!is_v) {
            if (is_k ? A.k_norm : A.q_norm) { /* for all rows of a kind */
                /* The sum goes over neighbours by pairs, in rows of more than 64 dimensions by fours in turn first, and no
                 * product is fused. Rows of 64, 128 and 256 dimensions then have the bits of the formula in elementary f32
                 * operations whose mean sums in that order, as torch's here does: a key's code, where a quotient lies on
                 * an edge, is the formula's. Other widths are summed as if zeros followed, and may differ by a rounding. */
                float q2[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    q2[i] = w[i] * w[i];
                float sum = LPR == 8 ? ((q2[0] + q2[1]) + (q2[2] + q2[3])) + ((q2[4] + q2[5]) + (q2[6] + q2[7]))
                                     : (((q2[0] + q2[1]) + q2[2]) + q2[3]) + (((q2[4] + q2[5]) + q2[6]) + q2[7]);
                sum = glint_add_dpp<GLINT_DPP_QUAD_1032>(sum);
                sum = glint_add_dpp<GLINT_DPP_QUAD_2301>(sum);
                sum = glint_add_dpp<GLINT_DPP_ROW_HALF_MIRROR>(sum);
                if constexpr (LPR >= 16)
                    sum = glint_add_dpp<GLINT_DPP_ROW_MIRROR>(sum);
                if constexpr (LPR >= 32)
                    sum += __shfl_xor(sum, 16, 64);
                const float r = kr_rsqrt(sum * A.inv_d + A.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    w[i] = w[i] * r * (is_k ? gk[i] : gq[i]);
            }
        }
        if (A.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                y[i] = w[i ^ 1];
        } else { /* every lane of the wave, also of rows that do not turn */
#pragma unroll
            for (int i = 0; i < 8; ++i)
                y[i] = __shfl(w[i], other, 64);
        }
        if (!is_v) {
            if (turned) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    w[i] = w[i] * cs[i] + y[i] * sn[i];
            }
            E *to = is_k ? (E *)A.k_out : (E *)A.q_out;
            if (live && to)
                kr_store8(to + (t * (is_k ? A.H : A.Hq) + h) * A.D + d, w);
        }
        if constexpr (CACHE) {
            if (row >= A.Hq) { /* of a row's 8 lanes, all or none */
                if constexpr (sizeof(E) == 2) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const uint32_t u = glint_cvt_bf16x2(w[i], w[i + 1]);
                        w[i] = glint_bf16lo(u);
                        w[i + 1] = glint_bf16hi(u);
                    }
                }
                float s;
                const uint32_t code = kt_code8<sizeof(E) == 2>(buckets, w, s);
                const int64_t ph = max(slot, (int64_t)0) / KV4_PAGE * A.H + h;
                const int at = (int)(slot & 63), e = c & 7, b = c >> 3;
                if (slot >= 0 && row < rows) {
                    if (is_v)
                        kt_put_value<KV4_PAGE>(A.v_hole + ph * (CD / 2 * KV4_PAGE) + at, 64 * b, e, code);
                    else
                        *(uint32_t *)(A.k_hole + (ph * KV4_PAGE + at) * (CD / 2) + kv4_k_byte<NB>(d)) = code;
                    if (e == 0)
                        (is_v ? A.v_absmax : A.k_absmax)[(ph * NB + b) * KV4_PAGE + at] = s;
                }
            }
        }
    }
}

/* Values go by tiles from where glint_kv4.hip's do. */
#define KR_TILE 6144 /* tokens of one head */
#define KR_TILE_T 16
/* Workgroups from which a token's rows are one workgroup's. */
#define KR_FULL 2048

template <class E, bool CACHE>
static int kr_launch(RotateArgs &a, hipStream_t stream) {
    const int lpr = CACHE ? a.D / 8 : a.D <= 64 ? 8 : a.D <= 128 ? 16 : 32;
    const int rows = a.Hq + a.H + a.value_rows, per = KR_T / lpr;
    a.parts = (rows + per - 1) / per;
    if (a.T >= KR_FULL)
        a.parts = 1;
    const int64_t grid = a.tiles + a.T * a.parts;
    if (grid > INT32_MAX / KR_T)
        return -2;
    const unsigned g = (unsigned)grid;
    if (lpr == 8)
        k_rotate<E, 8, CACHE><<<g, KR_T, 0, stream>>>(a);
    else if (lpr == 16)
        k_rotate<E, 16, CACHE><<<g, KR_T, 0, stream>>>(a);
    else if constexpr (!CACHE)
        k_rotate<E, 32, false><<<g, KR_T, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}

/* What both entry points refuse. */
static int kr_refuse(const RotateArgs &a, int elt, int norm_elt, int k_out_needed) {
    if (!a.q || !a.k || !a.pos || !a.freqs || !a.q_out || (k_out_needed && !a.k_out))
        return -1;
    if (elt != GLINT_KV_BF16 && elt != GLINT_KV_F32)
        return -2;
    if (a.T < 0 || a.T > (int64_t)1 << 31 || a.Hq < 1 || a.H < 1 || a.Hq > 65535 || a.H > 65535 || a.D < 16 || a.D > 256 ||
        a.D % 16 || a.rot < 16 || a.rot > a.D || a.rot % 16)
        return -2;
    if ((a.q_norm || a.k_norm) && norm_elt != GLINT_KV_BF16 && norm_elt != GLINT_KV_F32)
        return -2;
    const int64_t step = elt == GLINT_KV_BF16 ? 7 : 3;
    if (((a.q_st | a.q_sh | a.k_st | a.k_sh) & step) || !glint_aligned(a.q, 16) || !glint_aligned(a.k, 16) ||
        !glint_aligned(a.q_out, 16) || !glint_aligned(a.k_out, 16) || !glint_aligned(a.q_norm, 16) ||
        !glint_aligned(a.k_norm, 16))
        return -2;
    return 0;
}

GLINT_API int glint_rotate_qk(const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *k, int64_t k_stride_t,
                              int64_t k_stride_h, int elt, const int64_t *pos, const double *freqs, int64_t T, int Hq, int H,
                              int D, int rot, int interleaved, double magnitude, const void *q_norm, const void *k_norm,
                              int norm_elt, float eps, void *q_out, void *k_out, struct ihipStream_t *stream) {
    RotateArgs a{};
    a.q = q, a.q_st = q_stride_t, a.q_sh = q_stride_h;
    a.k = k, a.k_st = k_stride_t, a.k_sh = k_stride_h;
    a.pos = pos, a.freqs = freqs, a.T = T, a.Hq = Hq, a.H = H, a.D = D, a.rot = rot, a.interleaved = interleaved != 0;
    a.magnitude = magnitude, a.eps = eps, a.inv_d = 1.f / (float)D, a.q_norm = q_norm, a.k_norm = k_norm, a.norm_f32 = norm_elt == GLINT_KV_F32;
    a.q_out = q_out, a.k_out = k_out;
    const int rc = kr_refuse(a, elt, norm_elt, 1);
    if (rc || T == 0)
        return rc;
    return elt == GLINT_KV_BF16 ? kr_launch<uint16_t, false>(a, stream) : kr_launch<float, false>(a, stream);
}

GLINT_API int glint_kv4_append_rotated(const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *k,
                                       int64_t k_stride_t, int64_t k_stride_h, const void *v, int64_t v_stride_t,
                                       int64_t v_stride_h, int elt, const int64_t *pos, const double *freqs,
                                       const int64_t *slots, int64_t T, int Hq, int H, int D, int rot, int interleaved,
                                       double magnitude, const void *q_norm, const void *k_norm, int norm_elt, float eps,
                                       void *q_out, void *k_out, uint8_t *k_hole, float *k_absmax, uint8_t *v_hole,
                                       float *v_absmax, int64_t pages, struct ihipStream_t *stream) {
    RotateArgs a{};
    a.q = q, a.q_st = q_stride_t, a.q_sh = q_stride_h;
    a.k = k, a.k_st = k_stride_t, a.k_sh = k_stride_h;
    a.v = v, a.v_st = v_stride_t, a.v_sh = v_stride_h;
    a.pos = pos, a.freqs = freqs, a.T = T, a.Hq = Hq, a.H = H, a.D = D, a.rot = rot, a.interleaved = interleaved != 0;
    a.magnitude = magnitude, a.eps = eps, a.inv_d = 1.f / (float)D, a.q_norm = q_norm, a.k_norm = k_norm, a.norm_f32 = norm_elt == GLINT_KV_F32;
    a.q_out = q_out, a.k_out = k_out;
    a.slots = slots, a.k_hole = k_hole, a.k_absmax = k_absmax, a.v_hole = v_hole, a.v_absmax = v_absmax;
    a.nslots = pages * KV4_PAGE;
    if (!v || !slots || !k_hole || !k_absmax || !v_hole || !v_absmax)
        return -1;
    const int rc = kr_refuse(a, elt, norm_elt, 0);
    if (rc)
        return rc;
    if ((D != 64 && D != 128) || pages < 1 || pages >= (int64_t)1 << 40 || !glint_aligned(v, 16) ||
        ((v_stride_t | v_stride_h) & (elt == GLINT_KV_BF16 ? 7 : 3)) || !glint_aligned(k_hole, 16) ||
        !glint_aligned(v_hole, 16))
        return -2;
    if (T == 0)
        return 0;
    const bool tiles = T >= KR_TILE_T && T * H >= KR_TILE;
    const int64_t blocks = (T + KT_TOKENS - 1) / KT_TOKENS;
    if (tiles && blocks * H > INT32_MAX / KR_T)
        return -2;
    a.value_rows = tiles ? 0 : H;
    a.tile_blocks = (int)blocks;
    a.tiles = tiles ? (unsigned)(blocks * H) : 0;
    return elt == GLINT_KV_BF16 ? kr_launch<uint16_t, true>(a, stream) : kr_launch<float, true>(a, stream);
}
