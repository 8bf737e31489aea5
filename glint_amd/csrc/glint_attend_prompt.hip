/* Causal attention over packed prompts (include/glint_serve.h).
 *
 * k_attend_prompt — a workgroup of 4 waves takes 128 query rows of one head, 32 a wave, and
 *   walks the keys in tiles of 64 through LDS. Scores are formed transposed,
 *   S^T = K Q^T on the 32x32x16 bf16 matrix instruction, so that a lane holds 32 keys of one
 *   query row: maximum and sum are in-lane but for one exchange of the wave's halves, and the
 *   weights feed O^T = V^T P^T as they lie (the order of the keys inside a product is free).
 *   V^T operands come from the row-major V tile by the transposing LDS read.
 *
 *   One pass: each row keeps a running maximum m (in powers of two) and sum l = sum 2^(s - m), and its
 *   outputs are rescaled where m grows by more than AP_SLACK. Rounded to bf16: the weights (the
 *   matrix instruction's operand; what few large weights lose is added back) and the output.
 *
 *   What bounds it: 4 D operations a row and key on the matrix units and, beside them, some 12
 *   vector operations for a score. 8192 tokens, 32 heads of 128 over 8: 550 GFLOP in 535 to 572 us, 1.0
 *   PFLOP/s, where an 8192^3 product of the library reaches 1.2; of 64 dimensions, where a score's
 *   vector work is twice a product's share, 310 us. Four waves of 32 rows, two workgroups a CU
 *   (D = 128: 200 registers, 66 KB of LDS), so that one wave's exponentials run under
 *   another's products; loads a tile ahead, by the direct path to LDS, which needs no registers. A
 *   short prompt is bound by its longest row's tiles, one after another: 77 tokens 10 us. */
#include <algorithm>
#include <cfloat>
#include <cmath>

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
#define AP_STRIDE (1 << 24) /* elements: a tile's bytes fit 32 bits */
#define AP_SLACK 8.f /* a maximum may lag this far (in powers of two) before outputs are rescaled */

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
    int max_q, Hq, H, G;
    int nblk; /* row blocks of a head */
    int ngroups;
    uint32_t q_sign; /* 0x80008000 where the scale is negative */
    float scale2;    /* |scale| log2 e, above 0 */
    uint16_t *out;
};

/* Where 16-B chunk c of row r lies in an LDS tile's row: keys so that 8 lanes reading one
 * chunk of 8 rows touch 8 places, values so that the 64-B pieces of 4 rows that one transposing
 * read takes lie in different 64-B quarters of 256 B. */
__device__ __forceinline__ int ap_k_chunk(int r, int c) { return c ^ (r & 7); }
template <int D>
__device__ __forceinline__ int ap_v_chunk(int r, int c) { return D == 128 ? c ^ ((r & 3) << 2) : c ^ ((r & 2) << 1); }

typedef __attribute__((address_space(3))) char ap_lds;

/* 16 B per lane from the buffer to LDS at `to` + 16 lane (not in a template: the host pass refuses
 * the builtin where its arguments depend on one, and then leaves the kernel's stub out) */
__device__ __forceinline__ void ap_dma(__amdgpu_buffer_rsrc_t from, ap_lds *to, uint32_t offset, uint32_t more) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)to, 16, offset, more, 0, 0);
}

/* What a wave carries from tile to tile for its 32 rows. */
template <int D>
struct ApRows {
    ApFrag q[D / 16];
    ap_f32x16 o[D / 32];
    float m, l;
    int last;        /* this lane's row sees the keys up to here */
    uint32_t kat[4]; /* where the lane reads keys (by the chunk's low bits) and values (by dimension part) */
    uint32_t vat[D / 32];
};

/* One tile of keys. */
template <int D>
__device__ __forceinline__ void ap_tile(const ap_lds *kl, const ap_lds *vl, int t, ApRows<D> &w, float scale2, bool masked,
                                        int half) {
    ap_f32x16 sc[2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sc[a][i] = 0.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            ApFrag f;
            f.v = *(const __attribute__((address_space(3))) glint_u32x4 *)(kl + w.kat[s & 3] + 128 * (s >> 2) + a * 32 * D * 2);
            sc[a] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.f, w.q[s].f, sc[a], 0, 0, 0);
        }
    /* element i of part a is key 32 a + 8 (i / 4) + 4 half + i % 4 */
    if (masked) {
        const int first = t * AP_KEYS + 4 * half;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                sc[a][i] = first + 32 * a + 8 * (i >> 2) + (i & 3) <= w.last ? sc[a][i] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            top = fmaxf(top, sc[a][i]);
    top = glint_xor32(top, GlintMax()) * scale2;
    const bool more = top > w.m + AP_SLACK; /* a row's own test, here and below: its bits depend on no other row */
    if (__any(more)) {
        const float mn = more ? top : w.m;
        const float keep = __builtin_amdgcn_exp2f(w.m - (mn == -INFINITY ? 0.f : mn));
        w.m = mn;
        w.l *= keep;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                w.o[d][i] *= keep;
    }
    const float base = w.m == -INFINITY ? 0.f : w.m;
    ApFrag pf[4];
    float sum = 0.f;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
#pragma unroll
            for (int x = i; x < i + 2; ++x) {
                sc[a][x] = __builtin_amdgcn_exp2f(fmaf(sc[a][x], scale2, -base));
                sum += sc[a][x];
            }
            pf[2 * a + (i >> 3)].u[(i & 7) >> 1] = glint_cvt_bf16x2(sc[a][i], sc[a][i + 1]);
        }
    w.l += sum;
    /* Step s multiplies the keys that pf[s] holds: 16 s + 4 half + 0..3, and 8 on. */
    auto values = [&](int s, int d) {
        ApFrag f;
#pragma unroll
        for (int x = 0; x < 2; ++x)
            f.h[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ap_lds_s16x4 *)(vl + w.vat[d] + (16 * s + 8 * x) * D * 2));
        return f;
    };
    /* A weight's bf16 rounding (2^-8) averages out over many keys and does not where few hold
     * the sum: rows with a weight above 1 / 8 of their sum so far add what the rounding left. (8 equal
     * weights leave 2^-10.8 of a value's size, rms.) 12 packed prompts: 45.0 us without, 47.6 with 1 / 8,
     * 51.8 with 1 / 16; 8192 tokens 562, 565, 572. */
    const bool few = __builtin_amdgcn_exp2f(top - base) * 8.f > glint_xor32(w.l, GlintAdd());
    if (__any(few)) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            ApFrag rest;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int i = 8 * (s & 1) + 2 * x;
                const uint32_t left =
                    glint_cvt_bf16x2(sc[s >> 1][i] - glint_bf16lo(pf[s].u[x]), sc[s >> 1][i + 1] - glint_bf16hi(pf[s].u[x]));
                rest.u[x] = few ? left : 0u;
            }
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
                w.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(values(s, d).f, rest.f, w.o[d], 0, 0, 0);
        }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
            w.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(values(s, d).f, pf[s].f, w.o[d], 0, 0, 0);
}

template <int D>
__global__ __launch_bounds__(AP_T, D == 64 ? 4 : 2) void k_attend_prompt(ApArgs A) {
    constexpr int CH = D / 8;                  /* 16-B chunks of a row */
    constexpr int LOADS = AP_KEYS * CH / AP_T; /* of a thread, per tile of keys or values */
    constexpr int STEP = AP_T / CH;            /* rows that one load of every thread covers */
    constexpr int TILE = AP_KEYS * D * 2;      /* bytes */
    /* two tiles of each; arrays of their own, so that reads of one do not wait for loads into the other */
    __shared__ __attribute__((aligned(16))) char k0t[TILE], k1t[TILE], v0t[TILE], v1t[TILE];
    __shared__ uint32_t apart; /* a value that is not finite was taken out */
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    /* Work items are the row blocks of a group's heads, a group being one sequence and key head;
     * the longest rows come first. A workgroup's XCD is its index modulo 8, and each XCD's L2
     * should hold few groups' keys: as many groups as share out evenly go whole to one XCD
     * each; of the rest, where they divide 8, each goes to 8 / rest XCDs. 8192 tokens of 32
     * heads over 8 key heads: 555 us, 773 with every group on every XCD. What it costs: groups of
     * one XCD may be unlike, where a short sequence's heads fill the others. 4000 tokens and, in
     * the same call, prompts of 60 until the groups are 8: 4 key heads 153 us, the long one alone
     * 109; 2 key heads 148, 88; 1 key head 132, 86; 8 key heads (16 groups) 155, 163. */
    const int per = A.nblk * A.G, whole = A.ngroups & ~7, rest = A.ngroups & 7;
    int group, item;
    if ((int)blockIdx.x < whole * per) {
        const int on = (int)blockIdx.x >> 3;
        group = (on / per) * 8 + ((int)blockIdx.x & 7);
        item = on % per;
    } else {
        const int at = (int)blockIdx.x - whole * per;
        if (8 % rest == 0) {
            group = whole + (at & 7) % rest;
            item = (at >> 3) * (8 / rest) + (at & 7) / rest;
            if (item >= per)
                return;
        } else {
            group = whole + at % rest;
            item = at / rest;
        }
    }
    const int b = group / A.H, h = group % A.H, hq = h * A.G + item % A.G;
    const int64_t q0 = A.cu_q[b], k0 = A.cu_k[b];
    const int64_t q1 = A.cu_q[b + 1], k1 = A.cu_k[b + 1];
    if (q0 < 0 || q1 <= q0 || q1 > A.Tq)
        return;
    const int nq = (int)min(q1 - q0, (int64_t)A.max_q);
    const int nk = k0 >= 0 && k1 > k0 && k1 <= A.Tk ? (int)(k1 - k0) : 0;
    const int r0 = (A.nblk - 1 - item / A.G) * AP_ROWS;
    if (r0 >= nq)
        return;
    const int row = r0 + 32 * wave + col;
    const int64_t gap = nk - (q1 - q0); /* row i's last key is i + gap */
    /* the wave's first and last row's last keys: tiles up to the one need no mask, tiles past
     * the other nothing at all */
    const int wave_low = (int)max((int64_t)-1, r0 + 32 * wave + gap);
    const int wave_high = r0 + 32 * wave < nq ? (int)max((int64_t)-1, min(r0 + 32 * wave + 31, nq - 1) + gap) : -1;

    ApRows<D> w;
    w.m = -INFINITY;
    w.l = 0.f;
    w.last = row < nq ? (int)max((int64_t)-1, row + gap) : -1;
    {
        const uint16_t *qr = A.q + (q0 + min(row, nq - 1)) * A.q_st + hq * A.q_sh;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            w.q[s].v = *(const glint_u32x4 *)(qr + 16 * s + 8 * half);
#pragma unroll
            for (int x = 0; x < 4; ++x)
                w.q[s].u[x] ^= A.q_sign;
        }
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            w.o[d][i] = 0.f;
    /* Keys: row col (and col + 32), chunk 2 s + half. Values: a 16-lane group of the transposing
     * read takes 4 keys x 16 dimensions; lane i addresses key i / 4, dimensions 4 (i % 4), and
     * receives dimension i of the 4 keys. */
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w.kat[j] = col * D * 2 + 16 * ap_k_chunk(col, 2 * j + half);
    const int vkey = 4 * half + ((lane & 15) >> 2), vdim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
        w.vat[d] = vkey * D * 2 + 16 * ap_v_chunk<D>(vkey, (32 * d + vdim) >> 3) + 2 * (vdim & 7);

    const int64_t far = min(r0 + AP_ROWS, nq) - 1 + gap; /* the last key of the last row */
    const int ntiles = far < 0 ? 0 : (int)(far / AP_KEYS) + 1;
    const uint16_t *kb = A.k + k0 * A.k_st + h * A.k_sh, *vb = A.v + k0 * A.v_st + h * A.v_sh;

    /* Tiles go to LDS by the loads' direct path. Place p of a tile is chunk p % CH of row p / CH;
     * thread t fills places t + i AP_T, so its lane's global chunk carries the swizzle (the same
     * for every i). Rows past the sequence take an offset past the buffer's end: zeros. */
    const int my_row = threadIdx.x / CH, my_chunk = threadIdx.x % CH;
    const uint32_t ko = (uint32_t)(my_row * A.k_st * 2) + 16 * ap_k_chunk(my_row, my_chunk);
    const uint32_t vo = (uint32_t)(my_row * A.v_st * 2) + 16 * ap_v_chunk<D>(my_row, my_chunk);
    const uint32_t kstep = (uint32_t)(STEP * A.k_st * 2), vstep = (uint32_t)(STEP * A.v_st * 2);
    auto fetch = [&](int t, ap_lds *kt, ap_lds *vt) {
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void *)(kb + (int64_t)t * AP_KEYS * A.k_st),
                                                                            (short)0, 0x7FFFFFFF, GLINT_BUF_DWORD3);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void *)(vb + (int64_t)t * AP_KEYS * A.v_st),
                                                                            (short)0, 0x7FFFFFFF, GLINT_BUF_DWORD3);
        const int rows = nk - t * AP_KEYS;
        if (rows >= AP_KEYS) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                ap_dma(rk, kt + (i * AP_T + wave * 64) * 16, ko, i * kstep);
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                ap_dma(rv, vt + (i * AP_T + wave * 64) * 16, vo, i * vstep);
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const bool in = my_row + i * STEP < rows;
                ap_dma(rk, kt + (i * AP_T + wave * 64) * 16, in ? ko + i * kstep : 0xFFFFFF00u, 0);
                ap_dma(rv, vt + (i * AP_T + wave * 64) * 16, in ? vo + i * vstep : 0xFFFFFF00u, 0);
            }
        }
    };

    /* Of a tile that some row does not see whole, every thread looks through the values it loaded:
     * an infinite or NaN one, of which a weight of 0 would make NaN, becomes 0 until the
     * end. */
    const int t_part = (int)max((int64_t)0, r0 + gap + 1) / AP_KEYS;
    auto step = [&](int t, ap_lds *kt, ap_lds *vt, ap_lds *kn, ap_lds *vn) {
        __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0); /* this wave's part of tile t */
        __syncthreads();
        if (t + 1 < ntiles)
            fetch(t + 1, kn, vn); /* over tile t - 1, which every wave has left */
        if (t >= t_part) {
            typedef __attribute__((address_space(3))) glint_u32x4 lds_u32x4;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                lds_u32x4 *at = (lds_u32x4 *)(vt + (threadIdx.x + i * AP_T) * 16);
                glint_u32x4 x = *at;
                bool odd = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool lo = (x[j] & 0x7F80u) == 0x7F80u, hi = (x[j] & 0x7F800000u) == 0x7F800000u;
                    x[j] &= (lo ? 0xFFFF0000u : ~0u) & (hi ? 0xFFFFu : ~0u);
                    odd |= lo || hi;
                }
                if (odd) {
                    *at = x;
                    apart = 1;
                }
            }
            __syncthreads();
        }
        if (t * AP_KEYS <= wave_high)
            ap_tile<D>(kt, vt, t, w, A.scale2, t * AP_KEYS + AP_KEYS - 1 > wave_low, half);
    };
    if (threadIdx.x == 0)
        apart = 0;
    if (ntiles > 0)
        fetch(0, (ap_lds *)k0t, (ap_lds *)v0t);
    for (int t = 0; t < ntiles; t += 2) {
        step(t, (ap_lds *)k0t, (ap_lds *)v0t, (ap_lds *)k1t, (ap_lds *)v1t);
        if (t + 1 < ntiles)
            step(t + 1, (ap_lds *)k1t, (ap_lds *)v1t, (ap_lds *)k0t, (ap_lds *)v0t);
    }
    const float l = glint_xor32(w.l, GlintAdd());
    /* A value that is not finite leaves itself or NaN in its dimension of the rows that see it,
     * whatever its weight: the products above made NaN of some infinities, by what a weight's rounding
     * left (0, or negative), so the dimensions they spoilt are walked again for such values alone. */
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
        bool spoilt = false;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            spoilt |= !(fabsf(w.o[d][i]) <= FLT_MAX);
        if (!__any(spoilt && l <= FLT_MAX) && !__builtin_amdgcn_readfirstlane((int)apart))
            continue;
        ap_f32x16 odd;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            odd[i] = 0.f;
        for (int key = 0; key <= wave_high; ++key) {
            const uint16_t *from = vb + key * A.v_st + 32 * d + 4 * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t v = from[8 * (i >> 2) + (i & 3)];
                if ((v & 0x7F80u) == 0x7F80u && key <= w.last)
                    odd[i] += __uint_as_float(v << 16);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            w.o[d][i] = odd[i] == 0.f ? w.o[d][i] : odd[i];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    /* 8 dimensions in a lane once its halves have exchanged 4: 16-B stores */
    uint16_t *dst = A.out + ((q0 + min(row, nq - 1)) * A.Hq + hq) * D + 8 * half;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
            glint_u32x4 eight;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const auto two = __builtin_amdgcn_permlane32_swap(
                    glint_cvt_bf16x2(w.o[d][i + 2 * x] * inv, w.o[d][i + 2 * x + 1] * inv),
                    glint_cvt_bf16x2(w.o[d][i + 4 + 2 * x] * inv, w.o[d][i + 5 + 2 * x] * inv), false, false);
                eight[x] = two[0];
                eight[2 + x] = two[1];
            }
            if (row < nq)
                *(glint_u32x4 *)(dst + 32 * d + 2 * i) = eight;
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
    if (!glint_aligned(q, 16) || !glint_aligned(k, 16) || !glint_aligned(v, 16) || !glint_aligned(out, 16) ||
        ((q_stride_t | q_stride_h | k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7) || k_stride_t < D ||
        v_stride_t < D || k_stride_t > AP_STRIDE || v_stride_t > AP_STRIDE)
        return -2;
    if (B == 0 || Tq == 0 || max_q == 0)
        return 0;
    /* what one launch holds; max_q is a bound, so most row blocks of many sequences may be empty */
    const int nblk = (max_q + AP_ROWS - 1) / AP_ROWS;
    const int64_t most = (INT32_MAX / AP_T - 8) / ((int64_t)nblk * Hq); /* sequences */
    if (most < 1)
        return -2;
    const float scale2 = fabsf(scale) * 1.44269504088896341f;
    ApArgs a{q, k, v, q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h, cu_q, cu_k, Tq, Tk,
             max_q, Hq, H, Hq / H, nblk, 0, scale < 0.f ? 0x80008000u : 0u, scale2 < FLT_MIN ? FLT_MIN : scale2, out};
    const int per = a.nblk * a.G;
    for (int64_t b = 0; b < B; b += most) {
        a.cu_q = cu_q + b;
        a.cu_k = cu_k + b;
        a.ngroups = (int)std::min<int64_t>(B - b, most) * H;
        const int rest = a.ngroups & 7; /* 8 % rest == 0: whole rounds of 8 workgroups */
        const int tail = rest == 0 ? 0 : 8 % rest == 0 ? (per + 8 / rest - 1) / (8 / rest) * 8 : rest * per;
        const unsigned grid = (unsigned)((a.ngroups - rest) * per + tail);
        if (D == 64)
            k_attend_prompt<64><<<grid, AP_T, 0, stream>>>(a);
        else
            k_attend_prompt<128><<<grid, AP_T, 0, stream>>>(a);
        if (hipGetLastError() != hipSuccess)
            return -3;
    }
    return 0;
}
