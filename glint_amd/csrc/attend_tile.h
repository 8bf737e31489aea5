/* A tile of 64 keys under 32 query rows a wave: what the attention kernels over BF16 keys and values share. */
#ifndef GLINT_ATTEND_TILE_H_
#define GLINT_ATTEND_TILE_H_

#include "glint_common.h"

typedef __bf16 ap_bf16x8 __attribute__((ext_vector_type(8)));
typedef float ap_f32x16 __attribute__((ext_vector_type(16)));
typedef short ap_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ap_s16x4 ap_lds_s16x4;

#define AP_WAVES 4
#define AP_T (64 * AP_WAVES)
#define AP_ROWS (32 * AP_WAVES)
#define AP_KEYS 64
#define AP_SLACK 8.f /* a maximum may lag this far (in powers of two) before outputs are rescaled */

union ApFrag {
    uint32_t u[4];
    glint_u32x4 v;
    ap_s16x4 h[2];
    ap_bf16x8 f;
};

/* Where 16-B chunk c of row r lies in an LDS tile's row: keys so that 16 lanes reading one
 * chunk of 16 rows touch every bank once, values so that the 64-B pieces of 4 rows that one transposing
 * read takes lie in different 64-B quarters of 256 B. */
template <int D>
__device__ __forceinline__ int ap_k_chunk(int r, int c) { return c ^ (D == 128 ? r & 15 : (r >> 1) & 7); }
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

/* A row's bound: the last `window` positions up to its own, and the first `sinks`. */
struct ApBound {
    int window, sinks;
    __device__ bool sees(int key, int last) const { return key <= last && (key > last - window || key < sinks); }
};

/* One tile of keys, the first at position `at`. */
template <int D, bool BOUNDED>
__device__ __forceinline__ void ap_tile(const ap_lds *kl, const ap_lds *vl, int at, ApRows<D> &w, float scale2, bool masked,
                                        int half, const ApBound &bound) {
    ap_f32x16 sc[2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sc[a][i] = 0.f;
    /* Operands are read some products ahead; left to itself the compiler waits for the reads two by two. 8192 tokens of
     * 32 heads of 128 over 8: 542 us so, 533 with 4 ahead; 6 gain nothing more, and spill at D = 64. */
    constexpr int N = D / 8, AHEAD = 4;
    ApFrag f[AHEAD];
    auto read = [&](int n) {
        const int s = n >> 1, a = n & 1;
        f[n % AHEAD].v =
            *(const __attribute__((address_space(3))) glint_u32x4 *)(kl + (w.kat[s & 3] ^ (128 * (s >> 2))) + a * 32 * D * 2);
    };
#pragma unroll
    for (int n = 0; n < AHEAD; ++n)
        read(n);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        sc[n & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[n % AHEAD].f, w.q[n >> 1].f, sc[n & 1], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (n + AHEAD < N)
            read(n + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
    }
    /* element i of part a is key 32 a + 8 (i / 4) + 4 half + i % 4 */
    if (masked) {
        const int first = at + 4 * half;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = first + 32 * a + 8 * (i >> 2) + (i & 3);
                sc[a][i] = (BOUNDED ? bound.sees(key, w.last) : key <= w.last) ? sc[a][i] : -INFINITY;
            }
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

/* A row's outputs to dst, times inv: 8 dimensions in a lane once its halves have exchanged 4, 16-B stores. */
template <int D>
__device__ __forceinline__ void ap_store(uint16_t *dst, const ap_f32x16 (&o)[D / 32], float inv, int half, bool live) {
    dst += 8 * half;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
            glint_u32x4 eight;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const auto two = __builtin_amdgcn_permlane32_swap(
                    glint_cvt_bf16x2(o[d][i + 2 * x] * inv, o[d][i + 2 * x + 1] * inv),
                    glint_cvt_bf16x2(o[d][i + 4 + 2 * x] * inv, o[d][i + 5 + 2 * x] * inv), false, false);
                eight[x] = two[0];
                eight[2 + x] = two[1];
            }
            if (live)
                *(glint_u32x4 *)(dst + 32 * d + 2 * i) = eight;
        }
}

#endif
