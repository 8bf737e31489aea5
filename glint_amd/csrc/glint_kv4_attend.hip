/* Attention over the 4-bit cache (include/glint_serve.h).
 *
 * k_kv4_attend — the work is a list of rounds: a group is one sequence, key head and block of
 *   up to 16 NT query rows (the heads that share the key head, times the new tokens), and a
 *   round is KA_WAVES pages of a group, one a wave. Every workgroup takes an equal run of the
 *   list, whatever the lengths, so that a batch of short and long sequences fills the device
 *   evenly and the table below is filled once per workgroup. A wave keeps a running maximum,
 *   sum and output of its own; the waves meet in LDS at the end of a group, and the workgroups
 *   that share one in the last of them to arrive (partials in the stream's workspace, added in
 *   the groups' order, so the result does not depend on the arrival).
 *
 *   Per page of 64 tokens a wave forms scores transposed, S^T = K q^T, on
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
 */
#include <algorithm>

#include "kv4.h"
#include "tile_mfma.h"

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
#define KA_FAR (1 << 24) /* a page number past every sequence's: tables hold no more pages */

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
    float *part; /* two partials per workgroup; NULL: groups are not split */
    unsigned *ctr;
    int least; /* fewest rounds of a workgroup's run */
};

/* The sequence's rows and length, with every device value bounded. */
struct Kv4Seq {
    int64_t q0;
    int nq, rows, len, npages;
    int rounds; /* of a group; one at least: a group without pages writes zeros */
    int blocks; /* row blocks */
    int each;   /* units of a group: its rounds, or 1 where groups are not split */
    int units;  /* of the list that the sequence takes */
};
template <int COLS>
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttendArgs &a, int b) {
    Kv4Seq s;
    s.q0 = a.cu_q ? a.cu_q[b] : (int64_t)b * a.max_q;
    const int64_t q1 = a.cu_q ? a.cu_q[b + 1] : s.q0 + a.max_q;
    s.nq = s.q0 >= 0 && q1 > s.q0 && q1 <= a.Tq ? (int)(q1 - s.q0) : 0;
    s.rows = a.G * min(s.nq, a.max_q);
    s.len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * KV4_PAGE);
    s.npages = (s.len + KV4_PAGE - 1) / KV4_PAGE;
    s.rounds = max(1, (s.npages + KA_WAVES - 1) / KA_WAVES);
    s.blocks = (s.rows + COLS - 1) / COLS;
    s.each = a.part ? s.rounds : 1;
    s.units = s.each * s.blocks * a.H;
    return s;
}
__device__ __forceinline__ int kv4_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

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

/* A group, or the part of it that this workgroup's run holds. */
struct Kv4Group {
    Kv4Seq s;
    int b, at;       /* the sequence, and where in it the part begins */
    int h, rb;       /* key head, row block */
    int u, units;    /* place in the list, units */
    int begin, n;    /* first round, rounds */
};
/* A part that other workgroups share: what the one that joins them has to know. */
struct Kv4Join {
    int on, w_first, w_last, rows, rb, h;
    int64_t q0;
};

template <int D, int NT>
__global__ __launch_bounds__(KA_T) void k_kv4_attend(Kv4AttendArgs A) {
    constexpr int NB = D / 64, COLS = 16 * NT;
    constexpr int ROW = D + 4; /* a row's output, then its maximum and sum */
    __shared__ __attribute__((aligned(16))) uint32_t lds[KA_TABLE_WORDS];
    __shared__ __attribute__((aligned(16))) float meet[KA_WAVES * 16 * ROW];
    __shared__ __attribute__((aligned(16))) float scales[KA_WAVES * 2 * NB * KV4_PAGE];
    __shared__ unsigned s_last[2];

    const int lane = threadIdx.x & 63, wave = kv4_uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;

    /* this workgroup's run [u, u_end) of the list, and where it begins */
    const int per = (A.B + 63) / 64; /* sequences of a lane */
    int mine = 0;
    for (int i = 0; i < per; ++i)
        if (lane * per + i < A.B)
            mine += kv4_seq<COLS>(A, lane * per + i).units;
    int upto = mine;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const int v = __shfl_up(upto, k, 64);
        upto += lane >= k ? v : 0;
    }
    const int total = __builtin_amdgcn_readlane(upto, 63);
    const int share = max(A.least, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    if ((int64_t)blockIdx.x * share >= total)
        return;
    const int u_end = min(total - (int)blockIdx.x * share, share) + blockIdx.x * share;
    /* completes a group whose sequence, place in it and place in the list are set */
    auto place = [&](Kv4Group &G) {
        while (G.at >= G.s.units) { /* on to the sequence that it lies in */
            G.at -= G.s.units;
            G.s = kv4_seq<COLS>(A, ++G.b);
        }
        const int group = G.at / G.s.each;
        G.begin = G.at % G.s.each;
        G.h = kv4_uniform(group / G.s.blocks);
        G.rb = kv4_uniform(group % G.s.blocks);
        G.units = min(G.s.each - G.begin, u_end - G.u);
        G.n = A.part ? G.units : G.s.rounds;
    };
    Kv4Group G;
    {
        G.u = blockIdx.x * share;
        const int owner = __builtin_ctzll(__ballot(upto > G.u));
        G.at = G.u - __builtin_amdgcn_readlane(upto - mine, owner);
        G.b = owner * per;
        G.s = kv4_seq<COLS>(A, G.b);
        place(G);
    }

    const uint32_t lane4 = (uint32_t)(lane & (KA_COPIES - 1)) * 4;
    auto pair = [&](uint32_t word, int byte) { /* byte << 8 | lane4 */
        return *(const uint32_t *)((const char *)lds + __builtin_amdgcn_perm(word, lane4, 0x0C0C0000u | ((4u + byte) << 8)));
    };
    float *sl = scales + wave * (2 * NB * KV4_PAGE);

    /* This wave's pages of a group's part from its i-th round on, 64 of them, one a lane. A page
     * that is not there, past the sequence's end or not in the pool, is read as the pool's first
     * page and seen by nobody: its lane holds -1. */
    auto page_ids = [&](const Kv4Group &X, int i) {
        const int pg = (X.begin + i + lane) * KA_WAVES + wave;
        const int pid = i + lane < X.n && pg < X.s.npages ? A.table[X.b * A.table_stride + pg] : -1;
        return pid < A.pages ? pid : -1;
    };
    /* The lane's rows of q. */
    glint_u32x4 qw[NT][NB][2];
    auto load_q = [&](const Kv4Group &X) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = X.rb * COLS + 16 * n + col;
            const bool live = r < X.s.rows;
            const uint16_t *qr = A.q + (X.s.q0 + (live ? r / A.G : 0)) * A.q_st + (X.h * A.G + (live ? r % A.G : 0)) * A.q_sh;
#pragma unroll
            for (int bb = 0; bb < NB; ++bb)
#pragma unroll
                for (int st = 0; st < 2; ++st)
                    qw[n][bb][st] = *(const glint_u32x4 *)(qr + bb * 64 + 16 * g + 8 * st);
        }
    };
    /* A page's loads: this lane's 16-B pieces of the key rows and value columns, and one token's
     * scales, which go to the other lanes through LDS. `ph` is the page's place times the heads. */
    uint32_t kw[4][2 * NB];
    glint_u32x4 vw[D / 32];
    float sw[2 * NB];
    int64_t ph = 0;
    auto load_k = [&]() {
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
    auto load_v = [&]() {
        const uint8_t *vp = A.v_hole + ph * (KV4_PAGE * D / 2) + col * KV4_PAGE + 16 * g;
#pragma unroll
        for (int p = 0; p < D / 32; ++p)
            vw[p] = *(const glint_u32x4 *)(vp + p * (16 * KV4_PAGE));
    };
    int pids = page_ids(G, 0);
    auto page = [&](const Kv4Group &X, int i) { /* of round i; whether it is there */
        const int pid = __builtin_amdgcn_readlane(pids, i & 63);
        ph = (int64_t)max(pid, 0) * A.H + X.h;
        return pid >= 0;
    };
    load_q(G);
    for (int i = threadIdx.x; i < 256 * KA_COPIES / 4; i += KA_T) {
        const int byte = i / (KA_COPIES / 4);
        union {
            _Float16 f[2];
            uint32_t u;
        } e;
        e.f[0] = (_Float16)(kKv4Parent[byte & 15] * KA_ALPHA);
        e.f[1] = (_Float16)(kKv4Parent[byte >> 4] * KA_ALPHA);
        ((glint_u32x4 *)lds)[byte * 16 + i % (KA_COPIES / 4)] = glint_u32x4{e.u, e.u, e.u, e.u};
    }
    __syncthreads();
    bool there = page(G, 0);
    load_k();
    load_v();

    Kv4Join join0{0}, join1{0}; /* of this workgroup's slot 0 and slot 1 */
    while (true) {
    const Kv4Seq &s = G.s;
    /* the group after this one; its pages' numbers are on their way while this one's are read */
    Kv4Group N = G;
    N.u = G.u + G.units;
    N.at = G.at + G.units;
    const bool more_groups = N.u < u_end;
    int pids_next = -1;
    if (more_groups) {
        place(N);
        pids_next = page_ids(N, 0);
    }

    /* this lane's rows of q as f16 operands, scaled to 2^14 .. 2^15 by a power of two that goes
     * into the row's score factor */
    Kv4Frag qf[NT][NB][2];
    float factor[NT];
    int last[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = G.rb * COLS + 16 * n + col;
        last[n] = r < s.rows ? s.len - s.nq + r / A.G : -1;
        uint32_t top = 0;
#pragma unroll
        for (int bb = 0; bb < NB; ++bb)
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    top = max(top, max((qw[n][bb][st][x] & 0x7FFFu) << 16, qw[n][bb][st][x] & 0x7FFF0000u));
        top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
        const int ex = top >= 0x7F800000u ? 0 : (int)(top >> 23) - 127 - 14; /* 2^14 <= top 2^-ex < 2^15 */
#pragma unroll
        for (int bb = 0; bb < NB; ++bb)
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    qf[n][bb][st].f[2 * x] = (_Float16)ldexpf(glint_bf16lo(qw[n][bb][st][x]), -ex);
                    qf[n][bb][st].f[2 * x + 1] = (_Float16)ldexpf(glint_bf16hi(qw[n][bb][st][x]), -ex);
                }
        factor[n] = ldexpf(A.scale * (1.44269504088896341f / KA_ALPHA), ex);
    }

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

    for (int i = 0; i < G.n; ++i) {
        /* a page that nobody sees lies past every row's last position */
        const int pg = there ? (G.begin + i) * KA_WAVES + wave : KA_FAR;
        /* the run's last page is loaded again: without a branch around them the next page's
         * loads can be counted, and this page's waits leave them in flight */
        if (i + 1 < G.n) {
            /* waited for here, lest every page waits for its values where the branch joins */
            if (((i + 1) & 63) == 0) {
                pids = page_ids(G, i + 1);
                __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0);
            }
            there = page(G, i + 1);
        } else if (more_groups) {
            __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0);
            pids = pids_next;
            there = page(N, 0);
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
        load_k();
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
        load_v();
    }
    if (more_groups)
        load_q(N);

    /* The waves meet: each writes its rows' outputs, maximum and sum. A group that lies whole in
     * this workgroup's run is done; of one that does not, this workgroup's part goes to its slot
     * 1, where the group begins here, or 0. */
    const bool whole_group = G.n == s.rounds;
    const int slot = G.begin == 0;
    auto store = [&](int64_t q0, int h, int r, int d, const float (&acc)[4], float total) {
        const float inv = total == 0.f ? 0.f : 1.f / total;
        uint16_t *dst = A.out + ((q0 + r / A.G) * A.Hq + h * A.G + r % A.G) * D + d;
        glint_u32x2 two;
        two.x = glint_f32_to_bf16(acc[0] * inv) | (uint32_t)glint_f32_to_bf16(acc[1] * inv) << 16;
        two.y = glint_f32_to_bf16(acc[2] * inv) | (uint32_t)glint_f32_to_bf16(acc[3] * inv) << 16;
        *(glint_u32x2 *)dst = two;
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float sum = l[n];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        __syncthreads(); /* the previous rows are read */
        float *row = meet + (wave * 16 + col) * ROW;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            glint_f32x4 v = o[n][d];
            const float back = 1.f / vdown[n][d >> 2] * (1.f / KA_ALPHA); /* a power of two, inverted exactly */
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] *= back;
            *(glint_f32x4 *)(row + 16 * d + 4 * g) = v;
        }
        if (g == 0) {
            row[D] = m[n];
            row[D + 1] = sum;
        }
        __syncthreads();
        for (int t = threadIdx.x; t < 16 * (D / 4); t += KA_T) {
            const int c = t / (D / 4), d = 4 * (t % (D / 4));
            const int r = G.rb * COLS + 16 * n + c;
            if (r >= s.rows)
                continue;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < KA_WAVES; ++w)
                mx = fmaxf(mx, meet[(w * 16 + c) * ROW + D]);
            const float base = mx == -INFINITY ? 0.f : mx;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
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
            if (whole_group) {
                store(s.q0, G.h, r, d, acc, total);
            } else {
                float *dst = A.part + ((int64_t)(2 * blockIdx.x + slot) * COLS + 16 * n + c) * ROW;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    __hip_atomic_store(dst + d + i, acc[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (d == 0) {
                    __hip_atomic_store(dst + D, mx, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    __hip_atomic_store(dst + D + 1, total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
        }
    }
    if (!whole_group) {
        const int u_begin = G.u - G.begin;
        const Kv4Join J{1, u_begin / share, (u_begin + s.rounds - 1) / share, s.rows, G.rb, G.h, s.q0};
        if (slot)
            join1 = J;
        else
            join0 = J;
    }
    if (!more_groups)
        break;
    G = N;
    }

    /* The workgroups that share a group meet in the last of them to arrive: workgroup w_first has
     * its part in slot 1, those up to w_last in slot 0, and w_first's counter is theirs. */
    if (!join0.on && !join1.on)
        return;
    __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0);
    __syncthreads();
    auto arrive = [&](const Kv4Join &J) {
        return J.on && __hip_atomic_fetch_add(&A.ctr[J.w_first], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                           (unsigned)(J.w_last - J.w_first);
    };
    if (threadIdx.x == 0) {
        s_last[0] = arrive(join0);
        s_last[1] = arrive(join1);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const Kv4Join &J = j ? join1 : join0;
        if (!s_last[j])
            continue;
        for (int t = threadIdx.x; t < COLS * (D / 4); t += KA_T) {
            const int c = t / (D / 4), d = 4 * (t % (D / 4));
            const int r = J.rb * COLS + c;
            if (r >= J.rows)
                continue;
            float mx = -INFINITY, total = 0.f;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            for (int w0 = J.w_first; w0 <= J.w_last; w0 += 4) { /* four parts' loads in flight */
                float v[4][6];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int w = min(w0 + k, J.w_last);
                    const float *src = A.part + ((int64_t)(2 * w + (w == J.w_first)) * COLS + c) * ROW;
#pragma unroll
                    for (int i = 0; i < 6; ++i)
                        v[k][i] = __hip_atomic_load(src + (i < 4 ? d + i : D + i - 4), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (w0 + k <= J.w_last) {
                        const float to = fmaxf(mx, v[k][4]), base = to == -INFINITY ? 0.f : to;
                        const float keep = __builtin_amdgcn_exp2f(mx - base), f = __builtin_amdgcn_exp2f(v[k][4] - base);
                        mx = to;
                        total = fmaf(total, keep, f * v[k][5]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[i] = fmaf(acc[i], keep, f * v[k][i]);
                    }
            }
            const float inv = total == 0.f ? 0.f : 1.f / total;
            glint_u32x2 two;
            two.x = glint_f32_to_bf16(acc[0] * inv) | (uint32_t)glint_f32_to_bf16(acc[1] * inv) << 16;
            two.y = glint_f32_to_bf16(acc[2] * inv) | (uint32_t)glint_f32_to_bf16(acc[3] * inv) << 16;
            *(glint_u32x2 *)(A.out + ((J.q0 + r / A.G) * A.Hq + J.h * A.G + r % A.G) * D + d) = two;
        }
        if (threadIdx.x == 0)
            __hip_atomic_store(&A.ctr[J.w_first], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

/* Tiles of 16 rows a wave carries: two once a sequence's rows of a head fill more than one. */
static int ka_tiles(int max_q, int G) { return (int64_t)max_q * G > 16 ? 2 : 1; }

#ifndef KA_LEAST
#define KA_LEAST 2
#endif

static bool ka_shape(int B, int max_q, int Hq, int H, int D, int max_pages) {
    return B >= 0 && max_q >= 1 && H >= 1 && Hq >= H && Hq % H == 0 && (D == 64 || D == 128) && max_pages >= 1 &&
           max_pages <= KA_FAR && (int64_t)max_q * (Hq / H) <= (1 << 20);
}

/* Units of the longest list that the shape allows, or -1 where they leave 31 bits. */
static int64_t ka_units(int B, int max_q, int H, int G, int max_pages) {
    const int cols = 16 * ka_tiles(max_q, G);
    const int64_t blocks = ((int64_t)max_q * G + cols - 1) / cols, rounds = (max_pages + KA_WAVES - 1) / KA_WAVES;
    const double n = (double)B * H * (double)blocks * (double)rounds;
    return n > (double)(1 << 30) ? -1 : (int64_t)B * H * blocks * rounds;
}

template <int D, int NT>
static void ka_launch(const Kv4AttendArgs &a, int64_t units, hipStream_t stream) {
    const int64_t most = (units + a.least - 1) / a.least;
    k_kv4_attend<D, NT><<<(unsigned)std::min<int64_t>(most, glint_cu_count()), KA_T, 0, stream>>>(a);
}

GLINT_API int glint_serve_workspace_reserve(struct ihipStream_t *stream) {
    if (glint_stream_captures(stream))
        return -1;
    GlintSplitWs ws;
    return glint_split_ws_stream(stream, ws) ? 0 : -1;
}
GLINT_API int glint_serve_workspace_release(struct ihipStream_t *stream) { return glint_split_ws_release(stream); }

GLINT_API int glint_kv4_attend(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq,
                               const uint8_t *k_hole, const float *k_absmax, const uint8_t *v_hole,
                               const float *v_absmax, int64_t pages, const int32_t *table, int64_t table_stride,
                               int max_pages, const int32_t *lens, const int32_t *cu_q, int B, int max_q, int Hq, int H,
                               int D, float scale, uint16_t *out, struct ihipStream_t *stream) {
    if (!q || !k_hole || !k_absmax || !v_hole || !v_absmax || !table || !lens || !out)
        return -1;
    if (!ka_shape(B, max_q, Hq, H, D, max_pages) || Tq < 0 || pages < 1 || pages >= (int64_t)1 << 40 ||
        (!cu_q && Tq != (int64_t)B * max_q))
        return -2;
    if (!glint_aligned(q, 16) || !glint_aligned(out, 8) || !glint_aligned(k_hole, 16) || !glint_aligned(v_hole, 16) ||
        !glint_aligned(k_absmax, 16) || !glint_aligned(v_absmax, 16) || ((q_stride_t | q_stride_h) & 7))
        return -2;
    if (B == 0 || Tq == 0)
        return 0;
    Kv4AttendArgs a{q, q_stride_t, q_stride_h, Tq, k_hole, v_hole, k_absmax, v_absmax, pages, table, table_stride,
                    max_pages, lens, cu_q, B, max_q, Hq, H, Hq / H, scale, out, nullptr, nullptr, 1};
    int64_t units = ka_units(B, max_q, H, a.G, max_pages);
    if (units < 0)
        return -2;
    const bool two = ka_tiles(max_q, a.G) == 2;
    GlintSplitWs ws;
    if (max_pages > KA_WAVES && glint_split_ws_stream(stream, ws) && ws.nctr >= (size_t)glint_cu_count() &&
        ws.part_floats >= (size_t)glint_cu_count() * 2 * 32 * (D + 4)) {
        a.part = ws.part;
        a.ctr = ws.ctr;
        a.least = KA_LEAST;
    } else {
        units = ka_units(B, max_q, H, a.G, 1); /* whole groups */
    }
    if (D == 64)
        two ? ka_launch<64, 2>(a, units, stream) : ka_launch<64, 1>(a, units, stream);
    else
        two ? ka_launch<128, 2>(a, units, stream) : ka_launch<128, 1>(a, units, stream);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
