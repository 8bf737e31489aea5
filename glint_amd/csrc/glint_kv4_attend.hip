/* Attention over the 4-bit cache (include/glint_serve.h).
 *
 * k_kv4_attend — a workgroup takes a run of pages of one sequence and head for up to 16 NT
 *   query rows (the heads that share the key head, times the new tokens); its 8 waves take
 *   the run's pages in turn, each with a running maximum, sum and output of its own, and meet
 *   in LDS at the end. Per page of 64 tokens a wave forms scores transposed, S^T = K q^T, on
 *   the 16x16x32 f16 matrix instruction, so that a lane ends up with 16 tokens of one row,
 *   exponentiates in place and feeds them as they lie to O^T = V^T P^T: the order of the
 *   tokens inside a product is free, so the cache's rows are read in the order in which the
 *   first product leaves its results (token 16 g + 4 a + i for lane group g, tile a).
 *
 *   Codes become operands by a table in LDS: 256 entries, one per byte, the two f16 parents
 *   of its nibbles, in 32 copies so that a lane reads its own bank. A key byte holds
 *   adjacent dimensions, one operand register; a value byte holds dimensions 16 apart, two
 *   tiles' halves, and two tokens' entries are split by a byte permute.
 *
 *   Scales never touch the operands: a key's scale multiplies its 64-dimension partial score
 *   in f32, a value's is a factor of its softmax weight (one weight per 64 dimensions).
 *   f16 and not bf16: PARENT and the weights keep 11 bits and not 8, at the same rate. q
 *   (8 bits) fits f16 exactly once its row is scaled by a power of two; the weights are
 *   scaled by a power of two per row and 64-block that follows the largest value scale
 *   seen, so that they stay inside f16's range whatever the scales' size.
 *
 * k_kv4_join — adds the runs' outputs where a sequence was split over workgroups. */
#include <algorithm>

#include "kv4.h"

typedef _Float16 kv4_f16x8 __attribute__((ext_vector_type(8)));

#define KA_WAVES 8
#define KA_T (64 * KA_WAVES)
#define KA_COPIES 32 /* of an entry; entries are 64 words apart, so that an address is one byte permute */
#define KA_TABLE_WORDS (256 * 64)
/* The table holds PARENT * KA_ALPHA, whose f16 roundings are smaller and cancel: over the code
 * frequencies of normal values under a block-64 absmax (sigma 0.25 to 0.6 of it) and of even
 * ones, the mean error is at most 1.8e-6 of the absmax and the rms 3.9e-5, where PARENT's own
 * are 1.6e-5 and 9.5e-5. The mean counts: it is all that is left of the values' rounding in
 * the output of a long row, and at 8192 tokens of equal weight it alone was 0.8 of the bf16
 * output's rounding. */
#define KA_ALPHA 1.458935f
#define KA_VMAX 15 /* a scaled weight stays below 2^KA_VMAX */
#define KA_VSTART 10

union Kv4Frag {
    uint32_t u[4];
    kv4_f16x8 f;
};

struct Kv4AttendArgs {
    const uint16_t *q;
    int64_t q_st, q_sh, Tq;
    const uint8_t *k_hole, *v_hole;
    const float *k_absmax, *v_absmax;
    int64_t pages;
    const int32_t *table;
    int64_t table_stride;
    int max_pages;
    const int32_t *lens, *cu_q;
    int B, max_q, Hq, H, G;
    float scale;
    uint16_t *out;
    float *part;
    int nsplit, chunk; /* pages of a workgroup's run */
    int nrb;           /* row blocks of 16 NT */
};

/* The sequence's rows and length, with every device value bounded. */
struct Kv4Seq {
    int64_t q0;
    int nq, len, npages;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttendArgs &a, int b) {
    Kv4Seq s;
    s.q0 = a.cu_q ? a.cu_q[b] : (int64_t)b * a.max_q;
    const int64_t q1 = a.cu_q ? a.cu_q[b + 1] : s.q0 + a.max_q;
    s.nq = s.q0 >= 0 && q1 > s.q0 && q1 <= a.Tq ? (int)(q1 - s.q0) : 0;
    s.len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * KV4_PAGE);
    s.npages = (s.len + KV4_PAGE - 1) / KV4_PAGE;
    return s;
}

/* Some row's value scales leave f16's range: rows whose largest finite one does take a power
 * of two that puts it at 2^KA_VSTART and carry their outputs over. An infinite scale stays
 * infinite under any power and must not push the others out of range. */
template <int TILES>
__device__ __forceinline__ void kv4_new_power(const glint_f32x4 (&vscale)[4], float &down, float &limit, glint_f32x4 *o) {
    float top = 0.f;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            top = fmaxf(top, vscale[a][i] < INFINITY ? vscale[a][i] : 0.f);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (top < limit)
        return;
    const int e = max(-126, (int)(__float_as_uint(top) >> 23) - 127 - KA_VSTART);
    const float to = ldexpf(1.f, -e), by = to / down; /* by >= 2^-252: 0 where it underflows */
#pragma unroll
    for (int d = 0; d < TILES; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[d][i] *= by;
    down = to;
    limit = ldexpf(1.f, e + KA_VMAX);
}

template <int D, int NT>
__global__ __launch_bounds__(KA_T) void k_kv4_attend(Kv4AttendArgs A) {
    constexpr int NB = D / 64, COLS = 16 * NT;
    /* the table, then the waves' outputs over it: [wave][COLS][D + 4], m and l after each row */
    constexpr int ROW = D + 4;
    constexpr int LDS_WORDS = KA_WAVES * 16 * ROW > KA_TABLE_WORDS ? KA_WAVES * 16 * ROW : KA_TABLE_WORDS;
    __shared__ __attribute__((aligned(16))) uint32_t lds[LDS_WORDS];
    __shared__ __attribute__((aligned(16))) float scales[KA_WAVES * 2 * NB * KV4_PAGE];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int split = (int)blockIdx.x % A.nsplit, rb = (int)blockIdx.x / A.nsplit;
    const int h = blockIdx.y, b = blockIdx.z;
    const Kv4Seq s = kv4_seq(A, b);
    const int rows = A.G * min(s.nq, A.max_q);
    if (rb * COLS >= rows)
        return;
    const int p0 = split * A.chunk, p1 = min(p0 + A.chunk, s.npages);
    if (p0 >= p1 && split > 0)
        return;

    for (int i = threadIdx.x; i < 256 * KA_COPIES / 4; i += KA_T) {
        const int byte = i / (KA_COPIES / 4);
        union { _Float16 f[2]; uint32_t u; } e;
        e.f[0] = (_Float16)(kKv4Parent[byte & 15] * KA_ALPHA);
        e.f[1] = (_Float16)(kKv4Parent[byte >> 4] * KA_ALPHA);
        ((glint_u32x4 *)lds)[byte * 16 + i % (KA_COPIES / 4)] = glint_u32x4{e.u, e.u, e.u, e.u};
    }

    /* this lane's rows: q as f16 operands, scaled to 2^14 .. 2^15 by a power of two that goes
     * into the row's score factor */
    Kv4Frag qf[NT][NB][2];
    float factor[NT];
    int last[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = rb * COLS + 16 * n + col;
        const int i = r / A.G, hq = h * A.G + r % A.G;
        const bool live = r < rows;
        last[n] = live ? s.len - s.nq + i : -1;
        const uint16_t *qr = A.q + (s.q0 + (live ? i : 0)) * A.q_st + (live ? hq : h * A.G) * A.q_sh;
        glint_u32x4 w[NB][2];
        uint32_t top = 0;
#pragma unroll
        for (int bb = 0; bb < NB; ++bb)
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                w[bb][st] = *(const glint_u32x4 *)(qr + bb * 64 + 16 * g + 8 * st);
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    top = max(top, max((w[bb][st][x] & 0x7FFFu) << 16, w[bb][st][x] & 0x7FFF0000u));
            }
        top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
        const int ex = top >= 0x7F800000u ? 0 : (int)(top >> 23) - 127 - 14; /* 2^14 <= top 2^-ex < 2^15 */
#pragma unroll
        for (int bb = 0; bb < NB; ++bb)
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    qf[n][bb][st].f[2 * x] = (_Float16)ldexpf(glint_bf16lo(w[bb][st][x]), -ex);
                    qf[n][bb][st].f[2 * x + 1] = (_Float16)ldexpf(glint_bf16hi(w[bb][st][x]), -ex);
                }
        factor[n] = ldexpf(A.scale * (1.44269504088896341f / KA_ALPHA), ex);
    }
    __syncthreads();

    glint_f32x4 o[NT][D / 16];
    float m[NT], l[NT], vdown[NT][NB], vlimit[NT][NB];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            o[n][d] = glint_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int bb = 0; bb < NB; ++bb) {
            vdown[n][bb] = 0x1p126f;
            vlimit[n][bb] = 0x1p-111f;
        }
    }

    const uint32_t lane4 = (uint32_t)(lane & (KA_COPIES - 1)) * 4;
    auto pair = [&](uint32_t word, int byte) { /* byte << 8 | lane4 */
        return *(const uint32_t *)((const char *)lds + __builtin_amdgcn_perm(word, lane4, 0x0C0C0000u | ((4u + byte) << 8)));
    };

    /* A page's loads: this lane's 16-B pieces of the key rows and value columns, and one token's
     * scales, which go to the other lanes through LDS. */
    uint32_t kw[4][2 * NB];
    glint_u32x4 vw[D / 32];
    float sw[2 * NB];
    auto load_k = [&](int64_t ph) {
        const uint8_t *kp = A.k_hole + ph * (KV4_PAGE * D / 2) + (16 * (col >> 2) + (col & 3)) * (D / 2) + g * (8 * NB);
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int x = 0; x < 2 * NB; ++x)
                kw[a][x] = ((const uint32_t *)(kp + a * (4 * D / 2)))[x];
#pragma unroll
        for (int bb = 0; bb < NB; ++bb) {
            sw[bb] = A.k_absmax[ph * (NB * KV4_PAGE) + bb * KV4_PAGE + lane];
            sw[NB + bb] = A.v_absmax[ph * (NB * KV4_PAGE) + bb * KV4_PAGE + lane];
        }
    };
    auto load_v = [&](int64_t ph) {
        const uint8_t *vp = A.v_hole + ph * (KV4_PAGE * D / 2) + col * KV4_PAGE + 16 * g;
#pragma unroll
        for (int p = 0; p < D / 32; ++p)
            vw[p] = *(const glint_u32x4 *)(vp + p * (16 * KV4_PAGE));
    };
    float *sl = scales + wave * (2 * NB * KV4_PAGE);

    for (int pg0 = p0 + wave; pg0 < p1; pg0 += 64 * KA_WAVES) {
        /* this wave's next 64 pages, one a lane; those outside the pool drop out */
        const int mine = pg0 + lane * KA_WAVES;
        const int pid_mine = mine < p1 ? A.table[b * A.table_stride + mine] : -1;
        uint64_t todo = __ballot(pid_mine >= 0 && pid_mine < A.pages);
        if (todo == 0)
            continue;
        int at = __builtin_ctzll(todo);
        todo &= todo - 1;
        int64_t ph = (int64_t)__builtin_amdgcn_readlane(pid_mine, at) * A.H + h;
        load_k(ph);
        load_v(ph);
        for (bool more = true; more;) {
        const int pg = pg0 + at * KA_WAVES;
        more = todo != 0;
        if (more) {
            at = __builtin_ctzll(todo);
            todo &= todo - 1;
            ph = (int64_t)__builtin_amdgcn_readlane(pid_mine, at) * A.H + h;
        }
#pragma unroll
        for (int x = 0; x < 2 * NB; ++x)
            sl[x * KV4_PAGE + lane] = sw[x];

        /* scores */
        glint_f32x4 sc[NT][4];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            glint_f32x4 c[NT][NB];
#pragma unroll
            for (int bb = 0; bb < NB; ++bb) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    c[n][bb] = glint_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    Kv4Frag f;
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        f.u[x] = pair(kw[a][2 * bb + st], x);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        c[n][bb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.f, qf[n][bb][st].f, c[n][bb], 0, 0, 0);
                }
            }
            glint_f32x4 kscale[NB];
#pragma unroll
            for (int bb = 0; bb < NB; ++bb)
                kscale[bb] = *(const glint_f32x4 *)(sl + bb * KV4_PAGE + 16 * g + 4 * a);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = c[n][0][i] * kscale[0][i];
                    if (NB == 2)
                        x = fmaf(c[n][NB - 1][i], kscale[NB - 1][i], x);
                    sc[n][a][i] = x * factor[n];
                }
        }
        if (more)
            load_k(ph);
        /* what the row does not see; a whole page below every row's last position needs no look */
        const int t0 = pg * KV4_PAGE + 16 * g;
        const bool whole = (pg + 1) * KV4_PAGE <= s.len - s.nq + 1;
        if (!whole) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int a = 0; a < 4; ++a)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sc[n][a][i] = t0 + 4 * a + i <= last[n] ? sc[n][a][i] : -INFINITY;
        }

        /* softmax weights, times the value scales, as f16 */
        Kv4Frag pf[NT][NB][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float top = sc[n][0][0];
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    top = fmaxf(top, sc[n][a][i]);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any(top > m[n])) {
                const float mn = fmaxf(m[n], top);
                const float keep = __builtin_amdgcn_exp2f(m[n] - (mn == -INFINITY ? 0.f : mn));
                m[n] = mn;
                l[n] *= keep;
#pragma unroll
                for (int d = 0; d < D / 16; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[n][d][i] *= keep;
            }
            const float base = m[n] == -INFINITY ? 0.f : m[n];
            float sum = 0.f;
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[n][a][i] = __builtin_amdgcn_exp2f(sc[n][a][i] - base);
                    sum += sc[n][a][i];
                }
            l[n] += sum;
#pragma unroll
            for (int bb = 0; bb < NB; ++bb) {
                glint_f32x4 vscale[4];
                float vtop = 0.f;
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    vscale[a] = *(const glint_f32x4 *)(sl + (NB + bb) * KV4_PAGE + 16 * g + 4 * a);
                    if (!whole) { /* an unseen place counts as 0, whatever it holds */
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            vscale[a][i] = t0 + 4 * a + i <= last[n] ? vscale[a][i] : 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        vtop = fmaxf(vtop, vscale[a][i]);
                }
                if (__any(vtop >= vlimit[n][bb])) /* outside f16's range under some row's power */
                    kv4_new_power<D / (16 * NB)>(vscale, vdown[n][bb], vlimit[n][bb], &o[n][4 * bb]);
#pragma unroll
                for (int a = 0; a < 4; ++a)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        pf[n][bb][a >> 1].f[4 * (a & 1) + i] = (_Float16)(sc[n][a][i] * (vscale[a][i] * vdown[n][bb]));
            }
        }

        /* outputs */
#pragma unroll
        for (int p = 0; p < D / 32; ++p) {
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                Kv4Frag lo, hi;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t w = vw[p][2 * st + (x >> 1)];
                    const uint32_t e0 = pair(w, 2 * (x & 1)), e1 = pair(w, 2 * (x & 1) + 1);
                    lo.u[x] = __builtin_amdgcn_perm(e1, e0, 0x05040100u);
                    hi.u[x] = __builtin_amdgcn_perm(e1, e0, 0x07060302u);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    o[n][2 * p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo.f, pf[n][p >> 1][st].f, o[n][2 * p], 0, 0, 0);
                    o[n][2 * p + 1] =
                        __builtin_amdgcn_mfma_f32_16x16x32_f16(hi.f, pf[n][p >> 1][st].f, o[n][2 * p + 1], 0, 0, 0);
                }
            }
        }
        if (more)
            load_v(ph);
        }
    }

    /* the waves meet: each writes its rows' outputs, maximum and sum */
    float *meet = (float *)lds;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float sum = l[n];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        __syncthreads(); /* the table, or the previous rows, are read */
        float *row = meet + (wave * 16 + col) * ROW;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            glint_f32x4 v = o[n][d];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = v[i] / vdown[n][d >> 2] * (1.f / KA_ALPHA);
            *(glint_f32x4 *)(row + 16 * d + 4 * g) = v;
        }
        if (g == 0) {
            row[D] = m[n];
            row[D + 1] = sum;
        }
        __syncthreads();
        for (int t = threadIdx.x; t < 16 * (D / 4); t += KA_T) {
            const int c = t / (D / 4), d = 4 * (t % (D / 4));
            const int r = rb * COLS + 16 * n + c;
            if (r >= rows)
                continue;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < KA_WAVES; ++w)
                mx = fmaxf(mx, meet[(w * 16 + c) * ROW + D]);
            const float base = mx == -INFINITY ? 0.f : mx;
            glint_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            float total = 0.f;
#pragma unroll
            for (int w = 0; w < KA_WAVES; ++w) {
                const float *wr = meet + (w * 16 + c) * ROW;
                const float f = __builtin_amdgcn_exp2f(wr[D] - base);
                const glint_f32x4 v = *(const glint_f32x4 *)(wr + d);
                total = fmaf(f, wr[D + 1], total);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[i] = fmaf(f, v[i], acc[i]);
            }
            if (A.nsplit > 1) {
                float *dst = A.part + (((((int64_t)b * A.H + h) * A.nrb + rb) * A.nsplit + split) * COLS + 16 * n + c) * (D + 4);
                *(glint_f32x4 *)(dst + d) = acc;
                if (d == 0) {
                    dst[D] = mx;
                    dst[D + 1] = total;
                }
            } else {
                const float inv = total == 0.f ? 0.f : 1.f / total;
                uint16_t *dst = A.out + ((s.q0 + r / A.G) * A.Hq + h * A.G + r % A.G) * D + d;
                glint_u32x2 two;
                two.x = glint_f32_to_bf16(acc[0] * inv) | (uint32_t)glint_f32_to_bf16(acc[1] * inv) << 16;
                two.y = glint_f32_to_bf16(acc[2] * inv) | (uint32_t)glint_f32_to_bf16(acc[3] * inv) << 16;
                *(glint_u32x2 *)dst = two;
            }
        }
    }
}

/* One thread per 4 dimensions of a row: the runs that hold pages of the sequence (the first
 * one always writes), in order. */
template <int D, int NT>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4AttendArgs A) {
    constexpr int COLS = 16 * NT, PER = D / 4;
    const int h = blockIdx.y, b = blockIdx.z;
    const Kv4Seq s = kv4_seq(A, b);
    const int r = (int)((blockIdx.x * 256 + threadIdx.x) / PER), d = 4 * (int)(threadIdx.x % PER);
    if (r >= A.G * min(s.nq, A.max_q))
        return;
    const int used = max(1, (s.npages + A.chunk - 1) / A.chunk);
    const float *src = A.part + ((((int64_t)b * A.H + h) * A.nrb + r / COLS) * A.nsplit * COLS + r % COLS) * (D + 4);
    const int64_t step = (int64_t)COLS * (D + 4);
    float mx = -INFINITY;
    for (int i = 0; i < used; ++i)
        mx = fmaxf(mx, src[i * step + D]);
    const float base = mx == -INFINITY ? 0.f : mx;
    glint_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
    for (int i = 0; i < used; ++i) {
        const float f = __builtin_amdgcn_exp2f(src[i * step + D] - base);
        const glint_f32x4 v = *(const glint_f32x4 *)(src + i * step + d);
        total = fmaf(f, src[i * step + D + 1], total);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            acc[k] = fmaf(f, v[k], acc[k]);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    glint_u32x2 two;
    two.x = glint_f32_to_bf16(acc[0] * inv) | (uint32_t)glint_f32_to_bf16(acc[1] * inv) << 16;
    two.y = glint_f32_to_bf16(acc[2] * inv) | (uint32_t)glint_f32_to_bf16(acc[3] * inv) << 16;
    *(glint_u32x2 *)(A.out + ((s.q0 + r / A.G) * A.Hq + h * A.G + r % A.G) * D + d) = two;
}

/* Tiles of 16 rows a wave carries: two once a sequence's rows of a head fill more than one. */
static int ka_tiles(int max_q, int G) { return (int64_t)max_q * G > 16 ? 2 : 1; }

/* Runs of pages: enough workgroups for two per CU, none shorter than a page per wave. */
static void ka_plan(int B, int max_q, int Hq, int H, int max_pages, int &nrb, int &nsplit, int &chunk) {
    const int G = Hq / H, cols = 16 * ka_tiles(max_q, G);
    nrb = (int)(((int64_t)max_q * G + cols - 1) / cols);
    const int64_t groups = (int64_t)B * H * nrb, want = 2 * (int64_t)glint_cu_count();
    const int64_t most = max(1, (max_pages + KA_WAVES - 1) / KA_WAVES);
    const int64_t n = groups >= want ? 1 : std::min<int64_t>(most, (want + groups - 1) / groups);
    const int64_t per = (most + n - 1) / n; /* rounds of KA_WAVES pages */
    chunk = (int)(per * KA_WAVES);
    nsplit = (int)((most + per - 1) / per);
}

static bool ka_shape(int B, int max_q, int Hq, int H, int D, int max_pages) {
    return B >= 0 && B <= 65535 && max_q >= 1 && H >= 1 && H <= 65535 && Hq >= H && Hq % H == 0 &&
           (D == 64 || D == 128) && max_pages >= 1 && max_pages <= (1 << 25) && (int64_t)max_q * (Hq / H) <= (1 << 20);
}

GLINT_API int64_t glint_kv4_attend_part(int B, int max_q, int Hq, int H, int D, int max_pages) {
    if (!ka_shape(B, max_q, Hq, H, D, max_pages))
        return -2;
    int nrb, nsplit, chunk;
    ka_plan(B, max_q, Hq, H, max_pages, nrb, nsplit, chunk);
    return nsplit <= 1 ? 0 : (int64_t)B * H * nrb * nsplit * 16 * ka_tiles(max_q, Hq / H) * (D + 4);
}

template <int D, int NT>
static void ka_launch(const Kv4AttendArgs &a, hipStream_t stream) {
    k_kv4_attend<D, NT><<<dim3(a.nsplit * a.nrb, a.H, a.B), KA_T, 0, stream>>>(a);
    if (a.nsplit > 1) {
        const int per = 256 / (D / 4); /* rows per workgroup */
        k_kv4_join<D, NT><<<dim3((unsigned)((a.G * a.max_q + per - 1) / per), a.H, a.B), 256, 0, stream>>>(a);
    }
}

GLINT_API int glint_kv4_attend(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq,
                               const uint8_t *k_hole, const float *k_absmax, const uint8_t *v_hole,
                               const float *v_absmax, int64_t pages, const int32_t *table, int64_t table_stride,
                               int max_pages, const int32_t *lens, const int32_t *cu_q, int B, int max_q, int Hq, int H,
                               int D, float scale, uint16_t *out, float *part, struct ihipStream_t *stream) {
    if (!q || !k_hole || !k_absmax || !v_hole || !v_absmax || !table || !lens || !out)
        return -1;
    if (!ka_shape(B, max_q, Hq, H, D, max_pages) || Tq < 0 || pages < 1 || pages >= (int64_t)1 << 40 ||
        (!cu_q && Tq != (int64_t)B * max_q))
        return -2;
    if (!glint_aligned(q, 16) || !glint_aligned(out, 8) || !glint_aligned(k_hole, 16) || !glint_aligned(v_hole, 16) ||
        !glint_aligned(k_absmax, 16) || !glint_aligned(v_absmax, 16) || !glint_aligned(part, 16) ||
        ((q_stride_t | q_stride_h) & 7))
        return -2;
    if (B == 0 || Tq == 0)
        return 0;
    Kv4AttendArgs a{q, q_stride_t, q_stride_h, Tq, k_hole, v_hole, k_absmax, v_absmax, pages, table, table_stride,
                    max_pages, lens, cu_q, B, max_q, Hq, H, Hq / H, scale, out, part, 1, 1, 1};
    ka_plan(B, max_q, Hq, H, max_pages, a.nrb, a.nsplit, a.chunk);
    if (a.nsplit > 1 && !part)
        return -1;
    const bool two = ka_tiles(max_q, a.G) == 2;
    if (D == 64)
        two ? ka_launch<64, 2>(a, stream) : ka_launch<64, 1>(a, stream);
    else
        two ? ka_launch<128, 2>(a, stream) : ka_launch<128, 1>(a, stream);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
