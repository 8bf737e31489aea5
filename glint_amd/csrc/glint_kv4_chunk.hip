/* Attention of chunks of new tokens over the 4-bit cache (include/glint_serve.h).
 *
 * k_kv4_chunk — a group is one sequence, key head and block of up to 256 query rows (the heads that share
 *   the key head, times the new tokens), its work the tiles of 64 keys that its rows see: cached pages, then,
 *   where the call brings them, the new tokens' own keys. The groups' tiles form one list, and every
 *   workgroup takes an equal run of it, so that a long context under few rows fills the device and a ragged
 *   batch is shared out evenly. A workgroup keeps the maxima, sums and outputs of a group's rows (8 waves
 *   of 32) over its part; parts of one group meet in k_kv4_chunk_join.
 *
 *   A page is decoded once for all 256 rows: its codes become f16 operands by a table in LDS (one lookup a
 *   byte), times the row's scale, and lie there as K [64][D] and V^T [D][64], the next page's beside the one
 *   that is multiplied. V's tokens lie in the order in which the first product leaves its results (as
 *   attend_tile.h has it), so that both operands are plain 16-B reads. f16 and not bf16: PARENT, scales and
 *   weights keep 11 bits and not 8, at the same rate. Powers of two keep them in range: q's per row, the
 *   keys' and the values' per workgroup, following the largest scale seen. The new tokens' own keys and values
 *   are bf16 and go as in glint_attend_prompt.hip.
 *
 *   What bounds it: 4 D operations a row and key on the matrix units, the vector operations of a score beside
 *   them, and LDS, from which each wave reads every tile. */
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attend_tile.h"
#include "kv4.h"

typedef _Float16 kc_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 kc_f16x2 __attribute__((ext_vector_type(2)));

#define KC_WAVES 8
#define KC_T (64 * KC_WAVES)
#define KC_ROWS (32 * KC_WAVES)
#define KC_PAIRS 2048 /* of a sequence and a row block, in a launch */
#define KC_SHARE 2    /* tiles that a workgroup takes at least */
#define KC_UP 7.f     /* weights are 2^KC_UP times the softmax's: f16 has room above, and its small ones keep more bits */

struct KcArgs {
    const uint16_t *q;
    int64_t q_st, q_sh, Tq;
    const uint8_t *k_hole, *v_hole;
    const float *k_absmax, *v_absmax;
    int64_t pages;
    const int32_t *table;
    int64_t table_stride;
    int max_pages;
    const int32_t *lens, *cu_q;
    const uint16_t *k, *v; /* the new tokens' own, or NULL */
    int64_t k_st, k_sh, v_st, v_sh;
    int B, max_q, Hq, H, G, nblk;
    float scale2;    /* |scale| log2 e, above 0 */
    uint32_t q_sign; /* 0x80008000 where the scale is negative */
    uint16_t *out;
    ApBound bound;
    float *part;  /* outputs of two parts per workgroup, [KC_ROWS][D] each, */
    float *sums;  /* and their rows' maxima and sums */
};

/* A sequence; `held` of its positions are read from the cache, those from `own` on from k and v. */
struct KcSeq {
    int q0, nq, rows, len, held, own;
};
__device__ __forceinline__ KcSeq kc_seq(const KcArgs &a, int b) {
    KcSeq s{0, 0, 0, 0, 0, 0};
    const int64_t q0 = a.cu_q ? a.cu_q[b] : (int64_t)b * a.max_q, q1 = a.cu_q ? a.cu_q[b + 1] : q0 + a.max_q;
    if (q0 >= 0 && q1 > q0 && q1 <= a.Tq) {
        s.q0 = (int)q0;
        s.nq = (int)(q1 - q0);
        s.rows = a.G * min(s.nq, a.max_q);
    }
    const int most = (int)min((int64_t)INT32_MAX, (int64_t)a.max_pages * KV4_PAGE);
    s.len = max(a.lens[b], 0);
    if (a.k) {
        s.own = max(0, s.len - s.nq);
        s.held = min(s.own, most);
    } else {
        s.held = s.own = s.len = min(s.len, most);
    }
    return s;
}
/* The tiles of a row block: step i of the first np is page i, or, past the sinks', i + pskip; then nf tiles of own
 * keys likewise. */
struct KcTiles {
    int np, psinks, pskip, nf, fsinks, fskip;
};
__device__ __forceinline__ void kc_range(int upto, int64_t low, int64_t sinks, int &n, int &first, int &skip) {
    n = first = skip = 0;
    if (upto < 0)
        return;
    n = upto / AP_KEYS + 1;
    first = (int)((min(max(sinks, (int64_t)0), (int64_t)upto + 1) + AP_KEYS - 1) / AP_KEYS);
    skip = max(0, (int)min((int64_t)n, max(low, (int64_t)0) / AP_KEYS) - first);
    n -= skip;
}
__device__ __forceinline__ KcTiles kc_tiles(const KcArgs &a, const KcSeq &s, int rb) {
    KcTiles t{0, 0, 0, 0, 0, 0};
    if (rb * KC_ROWS >= s.rows)
        return t;
    const int p0 = s.len - s.nq + rb * KC_ROWS / a.G;
    const int p1 = s.len - s.nq + min(s.rows - 1, rb * KC_ROWS + KC_ROWS - 1) / a.G;
    const int64_t low = (int64_t)p0 - a.bound.window + 1;
    kc_range(min(s.held - 1, p1), low, a.bound.sinks, t.np, t.psinks, t.pskip);
    if (a.k)
        kc_range(p1 - s.own, low - s.own, (int64_t)a.bound.sinks - s.own, t.nf, t.fsinks, t.fskip);
    return t;
}
/* A row block that sees nothing counts as one tile: its rows are zero. */
__device__ __forceinline__ int kc_cost(const KcArgs &a, const KcSeq &s, int rb) {
    const KcTiles t = kc_tiles(a, s, rb);
    return rb * KC_ROWS < s.rows ? max(1, t.np + t.nf) : 0;
}

/* The list: sequences, of each its key heads, of each its row blocks. pre[i] is the cost of the pairs
 * (sequence, row block) before pair i. */
struct KcPlan {
    int pre[KC_PAIRS + 1];
    int wave[KC_WAVES];
    int b, rb, at;
};
__device__ __forceinline__ void kc_plan(const KcArgs &a, KcPlan &p) {
    const int pairs = a.B * a.nblk, per = (pairs + (int)blockDim.x - 1) / (int)blockDim.x, lane = threadIdx.x & 63;
    int mine[KC_PAIRS / 256], sum = 0;
    const int first = threadIdx.x * per;
#pragma unroll
    for (int i = 0; i < KC_PAIRS / 256; ++i) {
        mine[i] = 0;
        if (i < per && first + i < pairs)
            mine[i] = kc_cost(a, kc_seq(a, (first + i) / a.nblk), (first + i) % a.nblk);
        sum += mine[i];
    }
    int upto = sum;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const int v = __shfl_up(upto, step, 64);
        upto += lane >= step ? v : 0;
    }
    if (lane == 63)
        p.wave[threadIdx.x >> 6] = upto;
    __syncthreads();
    int before = upto - sum;
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w)
        before += p.wave[w];
#pragma unroll
    for (int i = 0; i < KC_PAIRS / 256; ++i) {
        if (i < per && first + i < pairs)
            p.pre[first + i] = before;
        before += mine[i];
        if (i < per && first + i == pairs - 1)
            p.pre[pairs] = before;
    }
    __syncthreads();
}
/* The group that unit u of the list lies in, and where in it. */
__device__ __forceinline__ void kc_find(const KcArgs &a, KcPlan &p, int u, int &b, int &h, int &rb, int &at) {
    for (int i = threadIdx.x; i < a.B; i += blockDim.x)
        if (a.H * p.pre[i * a.nblk] <= u && u < a.H * p.pre[(i + 1) * a.nblk])
            p.b = i;
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(p.b);
    const int *pre = p.pre + b * a.nblk;
    const int each = pre[a.nblk] - pre[0], in = u - a.H * pre[0];
    h = __builtin_amdgcn_readfirstlane(in / each);
    const int r = in % each + pre[0];
    for (int i = threadIdx.x; i < a.nblk; i += blockDim.x)
        if (pre[i] <= r && r < pre[i + 1]) {
            p.rb = i;
            p.at = r - pre[i];
        }
    __syncthreads();
    rb = __builtin_amdgcn_readfirstlane(p.rb);
    at = __builtin_amdgcn_readfirstlane(p.at);
}
__device__ __forceinline__ int kc_total(const KcArgs &a, const KcPlan &p) {
    return __builtin_amdgcn_readfirstlane(a.H * p.pre[a.B * a.nblk]);
}
__device__ __forceinline__ int kc_share(int total, int grid) { return max(KC_SHARE, (total + grid - 1) / grid); }

union KcFrag {
    uint32_t u[4];
    glint_u32x4 v;
    kc_f16x8 f;
    kc_f16x2 h[4];
};
__device__ __forceinline__ uint32_t kc_f16pair(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(glint_f32x2{lo, hi}, kc_f16x2));
}
__device__ __forceinline__ uint32_t kc_mul(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(kc_f16x2, a) * __builtin_bit_cast(kc_f16x2, b));
}

/* A power of two that follows scales up to `limit`. */
struct KcPower {
    float down = 0x1p126f, limit = 0x1p-111f;
    __device__ void follow(float v) { /* v of the wave's lanes, finite and not negative */
        if (!__any(v >= limit))
            return;
        const float top = glint_wave_max(v);
        const int e = max(-126, (int)(__float_as_uint(top) >> 23) - 127 - 14);
        down = ldexpf(1.f, -e);
        limit = ldexpf(1.f, e + 15);
    }
};

/* One page: as ap_tile, in f16, with the values' place the other way. `upto`: the last key that the lane's row
 * sees here. */
template <int D>
__device__ __forceinline__ void kc_tile(const ap_lds *kl, const ap_lds *vl, int at, ApRows<D> &w, const uint32_t (&vat)[4],
                                        float factor, bool masked, int upto, int half, const ApBound &bound) {
    typedef const __attribute__((address_space(3))) glint_u32x4 lds_u32x4;
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
            KcFrag f, q;
            f.v = *(lds_u32x4 *)(kl + w.kat[s & 3] + 128 * (s >> 2) + a * 32 * D * 2);
            q.v = w.q[s].v;
            sc[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.f, q.f, sc[a], 0, 0, 0);
        }
    if (masked) {
        const int first = at + 4 * half;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = first + 32 * a + 8 * (i >> 2) + (i & 3);
                sc[a][i] = key <= upto && bound.sees(key, w.last) ? sc[a][i] : -INFINITY;
            }
    }
    float top = -INFINITY;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            top = fmaxf(top, sc[a][i]);
    top = glint_xor32(top, GlintMax()) * factor;
    const bool more = top > w.m + AP_SLACK;
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
    const float base = w.m == -INFINITY ? 0.f : w.m - KC_UP;
    KcFrag pf[4];
    float sum = 0.f;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
#pragma unroll
            for (int x = i; x < i + 2; ++x) {
                sc[a][x] = __builtin_amdgcn_exp2f(fmaf(sc[a][x], factor, -base));
                sum += sc[a][x];
            }
            pf[2 * a + (i >> 3)].u[(i & 7) >> 1] = kc_f16pair(sc[a][i], sc[a][i + 1]);
        }
    w.l += sum;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
            KcFrag f;
            f.v = *(lds_u32x4 *)(vl + vat[s] + d * 32 * 128);
            w.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.f, pf[s].f, w.o[d], 0, 0, 0);
        }
}

template <int D>
__global__ __launch_bounds__(KC_T, 2) void k_kv4_chunk(KcArgs A) {
    constexpr int NB = D / 64, TILE = AP_KEYS * D * 2;
    constexpr int CH = D / 8, LOADS = AP_KEYS * CH / KC_T, STEP = KC_T / CH; /* of own keys, as in glint_attend_prompt.hip */
    /* codes' operands: byte, two f16 parents, in 32 copies; entries are 64 words apart, so that an address is one
     * byte permute */
    __shared__ __attribute__((aligned(16))) uint32_t entries[256 * 64];
    __shared__ __attribute__((aligned(16))) char k0t[TILE], k1t[TILE], v0t[TILE], v1t[TILE];
    __shared__ KcPlan plan;
    __shared__ uint32_t apart; /* a value that is not finite was taken out */

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    static_assert(KC_T == 512, "the table's shares: four copies of the entries t / 8 + 64 i");
    {
        const float lo = kKv4Parent[(threadIdx.x >> 3) & 15] * KV4_ALPHA;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t e = kc_f16pair(lo, kKv4Parent[(wave >> 1) + 4 * i] * KV4_ALPHA);
            ((glint_u32x4 *)entries)[((threadIdx.x >> 3) + 64 * i) * 16 + (threadIdx.x & 7)] = glint_u32x4{e, e, e, e};
        }
    }
    kc_plan(A, plan);
    const int grid = gridDim.x, total = kc_total(A, plan), share = kc_share(total, grid);
    /* neighbours in the list share keys: they go to one XCD, a workgroup's being its index modulo 8 */
    const int me = grid & 7 ? (int)blockIdx.x : ((int)blockIdx.x & 7) * (grid >> 3) + ((int)blockIdx.x >> 3);
    if ((int64_t)me * share >= total)
        return;
    int left = min(share, total - me * share); /* of this workgroup's run */
    int b, h, rb, at;
    kc_find(A, plan, me * share, b, h, rb, at);

    const uint32_t lane4 = (uint32_t)(lane & 31) * 4;
    auto pair = [&](uint32_t word, int byte) {
        return *(const uint32_t *)((const char *)entries + __builtin_amdgcn_perm(word, lane4, 0x0C0C0000u | ((4u + byte) << 8)));
    };
    ApRows<D> w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w.kat[j] = col * D * 2 + 16 * ap_k_chunk(col, 2 * j + half);
    uint32_t vat[4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
        vat[s] = col * 128 + 16 * ((2 * s + half) ^ (col & 7));
    const int vkey = 4 * half + ((lane & 15) >> 2), vdim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
        w.vat[d] = vkey * D * 2 + 16 * ap_v_chunk<D>(vkey, (32 * d + vdim) >> 3) + 2 * (vdim & 7);
    /* The thread's part of a page. Of the keys: NB words of the row of token ktok, dimensions 64 kb + 16 kc
     * (and 8 on where NB is 1 and the part odd). Of the values: row vrow, tokens vtok .. + 3 and, where NB is 2, 8 on. */
    const int kpart = threadIdx.x & 7, ktok = threadIdx.x >> 3;
    const int kb = NB == 2 ? kpart & 1 : 0;
    const int kdim = NB == 2 ? 64 * kb + 16 * (kpart >> 1) : 8 * kpart;
    const int vrow = NB == 2 ? threadIdx.x >> 3 : threadIdx.x >> 4;
    const int vtok = NB == 2 ? 16 * ((threadIdx.x & 7) >> 1) + 4 * (threadIdx.x & 1) : 4 * (threadIdx.x & 15);
    const int vhigh = ((vrow >> 4) << 5) + (vrow & 15); /* the low nibbles' dimension; the high ones' is 16 on */
    const uint32_t vto = vhigh * 128 + 16 * ((2 * (vtok >> 4) + ((vtok >> 2) & 1)) ^ (vhigh & 7)) + ((vtok >> 3) & 1) * 8;

    for (;;) {
        const KcSeq s = kc_seq(A, b);
        const KcTiles tiles = kc_tiles(A, s, rb);
        const int n = tiles.np + tiles.nf, cost = max(1, n);
        const int take = min(left, cost - at), end = min(at + take, n); /* tiles at .. end - 1 */
        const int row = rb * KC_ROWS + 32 * wave + col;
        const bool live = row < s.rows, wave_live = rb * KC_ROWS + 32 * wave < s.rows;
        const int gap = s.len - s.nq;
        const int wave_low = gap + (rb * KC_ROWS + 32 * wave) / A.G;
        const int wave_high = gap + min(s.rows - 1, rb * KC_ROWS + 32 * wave + 31) / A.G;
        const uint16_t *qr = A.q + (int64_t)(s.q0 + (live ? row / A.G : 0)) * A.q_st + (h * A.G + (live ? row % A.G : 0)) * A.q_sh;
        w.m = -INFINITY;
        w.l = 0.f;
        w.last = live ? gap + row / A.G : -1;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                w.o[d][i] = 0.f;
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
            w.q[x].v = *(const glint_u32x4 *)(qr + 16 * x + 8 * half);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w.q[x].u[i] ^= A.q_sign;
        }
        if (threadIdx.x == 0)
            apart = 0;
        /* whether a wave sees any, and all, of the keys at .. at + 63, as far as the window goes */
        auto bound_any = [&](int key) { return key + AP_KEYS - 1 > wave_low - A.bound.window || key < A.bound.sinks; };
        auto bound_all = [&](int key) { return key > wave_high - A.bound.window || key + AP_KEYS <= A.bound.sinks; };

        /* ---------------------------------------------------------------- cached pages */
        const int pend = min(end, tiles.np);
        if (at < pend) {
            const int32_t *pages = A.table + (int64_t)b * A.table_stride;
            auto page_of = [&](int i) { return i < tiles.psinks ? i : i + tiles.pskip; };
            /* q as f16, scaled to 2^14 .. 2^15 by a power of two of the row's */
            uint32_t high = 0;
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    high = max(high, max((w.q[x].u[i] & 0x7FFFu) << 16, w.q[x].u[i] & 0x7FFF0000u));
            high = __float_as_uint(glint_xor32(__uint_as_float(min(high, 0x7F800000u)), GlintMax()));
            const int ex = high >= 0x7F800000u ? 0 : (int)(high >> 23) - 127 - 14;
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w.q[x].u[i] = kc_f16pair(ldexpf(glint_bf16lo(w.q[x].u[i]), -ex), ldexpf(glint_bf16hi(w.q[x].u[i]), -ex));
            const float factor = ldexpf(A.scale2 / KV4_ALPHA, ex);
            const int upto = min(w.last, s.held - 1);
            /* what some row of the block sees; other places may hold anything */
            const int block_low = gap + rb * KC_ROWS / A.G - A.bound.window + 1;
            const int block_high = min(s.held - 1, gap + min(s.rows - 1, rb * KC_ROWS + KC_ROWS - 1) / A.G);
            auto seen = [&](int key) { return key <= block_high && (key >= block_low || key < A.bound.sinks); };

            /* the next 64 pages' numbers, one a lane; -1 where there is none */
            int window = at, pids;
            auto open_window = [&](int i) {
                window = i;
                pids = i + lane < pend ? pages[page_of(i + lane)] : -1;
                pids = pids < A.pages ? pids : -1;
            };
            open_window(at);
            uint32_t kw[NB], vw[NB];
            float ks, kall[NB], vall[NB];
            glint_f32x4 vs[NB];
            auto load = [&](int i) { /* whether the page is there */
                if (i - window == 64)
                    open_window(i);
                const int pid = __builtin_amdgcn_readlane(pids, i - window);
                const int64_t ph = (int64_t)max(pid, 0) * A.H + h;
                const uint8_t *kp = A.k_hole + ph * (KV4_PAGE * D / 2) + ktok * (D / 2) + kpart * (4 * NB);
                const uint8_t *vp = A.v_hole + ph * (KV4_PAGE * D / 2) + vrow * KV4_PAGE + vtok;
                const float *ka = A.k_absmax + ph * (NB * KV4_PAGE), *va = A.v_absmax + ph * (NB * KV4_PAGE);
                if constexpr (NB == 2) {
                    const glint_u32x2 two = *(const glint_u32x2 *)kp;
                    kw[0] = two.x;
                    kw[1] = two.y;
                } else {
                    kw[0] = *(const uint32_t *)kp;
                }
#pragma unroll
                for (int x = 0; x < NB; ++x) {
                    vw[x] = *(const uint32_t *)(vp + 8 * x);
                    vs[x] = *(const glint_f32x4 *)(va + (vhigh >> 6) * KV4_PAGE + vtok + 8 * x);
                    kall[x] = ka[x * KV4_PAGE + lane];
                    vall[x] = va[x * KV4_PAGE + lane];
                }
                ks = ka[kb * KV4_PAGE + ktok];
                return pid >= 0;
            };
            KcPower kpow, vpow;
            float odown = vpow.down; /* the power that the outputs so far have */
            auto decode = [&](int i, bool there, ap_lds *kt, ap_lds *vt) {
                if (!there)
                    return;
                const int key = page_of(i) * KV4_PAGE;
                float km = 0.f, vm = 0.f;
                bool odd = false;
#pragma unroll
                for (int x = 0; x < NB; ++x) {
                    const float ak = fabsf(kall[x]), av = fabsf(vall[x]);
                    km = ak <= FLT_MAX ? fmaxf(km, ak) : km;
                    vm = av <= FLT_MAX ? fmaxf(vm, av) : vm;
                    odd |= !(av <= FLT_MAX);
                }
                const bool in = seen(key + lane);
                odd &= in;
                if (odd)
                    apart = 1;
                const bool all = __all(in && !odd);
                kpow.follow(in ? km : 0.f);
                vpow.follow(in ? vm : 0.f);
                /* keys */
                const uint32_t k2 = kc_f16pair(ks * kpow.down, ks * kpow.down);
                typedef __attribute__((address_space(3))) glint_u32x4 lds_u32x4;
                typedef __attribute__((address_space(3))) glint_u32x2 lds_u32x2;
#pragma unroll
                for (int x = 0; x < NB; ++x) {
                    glint_u32x4 eight;
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        eight[y] = kc_mul(pair(kw[x], y), k2);
                    *(lds_u32x4 *)(kt + ktok * (D * 2) + 16 * ap_k_chunk(ktok, kdim / 8 + x)) = eight;
                }
                /* values */
                glint_u32x2 lo[NB], hi[NB];
#pragma unroll
                for (int x = 0; x < NB; ++x) {
                    float f[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        f[y] = vs[x][y] * vpow.down;
                    if (!all) {
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            f[y] = fabsf(vs[x][y]) <= FLT_MAX && seen(key + vtok + 8 * x + y) ? f[y] : 0.f;
                    }
                    uint32_t e[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        e[y] = pair(vw[x], y);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint32_t sc = kc_f16pair(f[2 * y], f[2 * y + 1]);
                        lo[x][y] = kc_mul(__builtin_amdgcn_perm(e[2 * y + 1], e[2 * y], 0x05040100u), sc);
                        hi[x][y] = kc_mul(__builtin_amdgcn_perm(e[2 * y + 1], e[2 * y], 0x07060302u), sc);
                    }
                }
                if constexpr (NB == 2) {
                    *(lds_u32x4 *)(vt + vto) = glint_u32x4{lo[0].x, lo[0].y, lo[1].x, lo[1].y};
                    *(lds_u32x4 *)(vt + vto + 16 * 128) = glint_u32x4{hi[0].x, hi[0].y, hi[1].x, hi[1].y};
                } else {
                    *(lds_u32x2 *)(vt + vto) = lo[0];
                    *(lds_u32x2 *)(vt + vto + 16 * 128) = hi[0];
                }
            };
            bool there = load(at);
            __syncthreads(); /* the table is written, the last group's tiles are read, apart is cleared */
            decode(at, there, (ap_lds *)k0t, (ap_lds *)v0t);
            __syncthreads();
            auto step = [&](int i, ap_lds *kt, ap_lds *vt, ap_lds *kn, ap_lds *vn) {
                const bool now = there;
                const float vdown = vpow.down, f = fminf(fmaxf(factor / kpow.down, FLT_MIN), FLT_MAX);
                const bool more = i + 1 < pend;
                if (more)
                    there = load(i + 1);
                const int key = page_of(i) * KV4_PAGE;
                if (now && wave_live && key <= min(wave_high, s.held - 1) && bound_any(key)) {
                    if (vdown != odown) {
                        const float by = vdown / odown;
#pragma unroll
                        for (int d = 0; d < D / 32; ++d)
#pragma unroll
                            for (int x = 0; x < 16; ++x)
                                w.o[d][x] *= by;
                        odown = vdown;
                    }
                    kc_tile<D>(kt, vt, key, w, vat, f, key + AP_KEYS - 1 > min(wave_low, s.held - 1) || !bound_all(key), upto,
                               half, A.bound);
                }
                if (more)
                    decode(i + 1, there, kn, vn);
                __syncthreads();
            };
            for (int i = at; i < pend; i += 2) {
                step(i, (ap_lds *)k0t, (ap_lds *)v0t, (ap_lds *)k1t, (ap_lds *)v1t);
                if (i + 1 < pend)
                    step(i + 1, (ap_lds *)k1t, (ap_lds *)v1t, (ap_lds *)k0t, (ap_lds *)v0t);
            }
            const float back = 1.f / odown * (1.f / KV4_ALPHA) * 0x1p-7f;
            w.l *= 0x1p-7f;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    w.o[d][x] *= back;
        }

        /* ---------------------------------------------------------------- own keys */
        const int f0 = max(at - tiles.np, 0), f1 = end - tiles.np;
        const int64_t own_row = (int64_t)s.q0 + s.nq - s.len; /* the row of k and v of position 0 */
        if (f0 < f1) {
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
                w.q[x].v = *(const glint_u32x4 *)(qr + 16 * x + 8 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w.q[x].u[i] ^= A.q_sign;
            }
            auto tile_of = [&](int i) { return i < tiles.fsinks ? i : i + tiles.fskip; };
            const uint16_t *k0 = A.k + (own_row + s.own) * A.k_st + h * A.k_sh, *v0 = A.v + (own_row + s.own) * A.v_st + h * A.v_sh;
            const int my_row = threadIdx.x / CH, my_chunk = threadIdx.x % CH;
            const uint32_t ko = (uint32_t)(my_row * A.k_st * 2) + 16 * ap_k_chunk(my_row, my_chunk);
            const uint32_t vo = (uint32_t)(my_row * A.v_st * 2) + 16 * ap_v_chunk<D>(my_row, my_chunk);
            const uint32_t kstep = (uint32_t)(STEP * A.k_st * 2), vstep = (uint32_t)(STEP * A.v_st * 2);
            auto fetch = [&](int t, ap_lds *kt, ap_lds *vt) { /* rows past the sequence: zeros */
                const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
                    (void *)(k0 + (int64_t)t * AP_KEYS * A.k_st), (short)0, 0x7FFFFFFF, GLINT_BUF_DWORD3);
                const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
                    (void *)(v0 + (int64_t)t * AP_KEYS * A.v_st), (short)0, 0x7FFFFFFF, GLINT_BUF_DWORD3);
                const int rows = s.len - s.own - t * AP_KEYS;
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const bool in = my_row + i * STEP < rows;
                    ap_dma(rk, kt + (i * KC_T + wave * 64) * 16, in ? ko + i * kstep : 0xFFFFFF00u, 0);
                    ap_dma(rv, vt + (i * KC_T + wave * 64) * 16, in ? vo + i * vstep : 0xFFFFFF00u, 0);
                }
            };
            auto step = [&](int i, ap_lds *kt, ap_lds *vt, ap_lds *kn, ap_lds *vn) {
                const int key = s.own + tile_of(i) * AP_KEYS;
                __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0);
                __syncthreads();
                if (i + 1 < f1)
                    fetch(tile_of(i + 1), kn, vn);
                /* an infinite or NaN value, of which a weight of 0 would make NaN, becomes 0 until the end */
                typedef __attribute__((address_space(3))) glint_u32x4 lds_u32x4;
#pragma unroll
                for (int x = 0; x < LOADS; ++x) {
                    lds_u32x4 *place = (lds_u32x4 *)(vt + (threadIdx.x + x * KC_T) * 16);
                    glint_u32x4 e = *place;
                    bool odd = false;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool lo = (e[j] & 0x7F80u) == 0x7F80u, hi = (e[j] & 0x7F800000u) == 0x7F800000u;
                        e[j] &= (lo ? 0xFFFF0000u : ~0u) & (hi ? 0xFFFFu : ~0u);
                        odd |= lo || hi;
                    }
                    if (odd) {
                        *place = e;
                        apart = 1;
                    }
                }
                __syncthreads();
                if (wave_live && key <= wave_high && bound_any(key))
                    ap_tile<D, true>(kt, vt, key, w, A.scale2, key + AP_KEYS - 1 > wave_low || !bound_all(key), half, A.bound);
            };
            __syncthreads(); /* the last tiles are read, apart is cleared */
            fetch(tile_of(f0), (ap_lds *)k0t, (ap_lds *)v0t);
            for (int i = f0; i < f1; i += 2) {
                step(i, (ap_lds *)k0t, (ap_lds *)v0t, (ap_lds *)k1t, (ap_lds *)v1t);
                if (i + 1 < f1)
                    step(i + 1, (ap_lds *)k1t, (ap_lds *)v1t, (ap_lds *)k0t, (ap_lds *)v0t);
            }
        }

        /* A value that is not finite leaves itself or NaN in its dimension of the rows that see it, whatever its
         * weight. */
        __syncthreads();
        const bool spoilt = __builtin_amdgcn_readfirstlane((int)apart);
        __syncthreads(); /* before the next group clears it */
        if (spoilt) {
#pragma unroll 1
            for (int d = 0; d < D / 32; ++d) {
                ap_f32x16 odd;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    odd[i] = 0.f;
                for (int i = at; i < pend; ++i) {
                    const int page = i < tiles.psinks ? i : i + tiles.pskip;
                    const int pid = A.table[(int64_t)b * A.table_stride + page];
                    if (pid < 0 || pid >= A.pages)
                        continue;
                    const int64_t ph = (int64_t)pid * A.H + h;
                    const float sv = A.v_absmax[ph * (NB * KV4_PAGE) + (d >> 1) * KV4_PAGE + lane];
                    uint64_t hit = __ballot(!(fabsf(sv) <= FLT_MAX) && page * KV4_PAGE + lane < s.held);
                    for (; hit; hit &= hit - 1) {
                        const int j = __builtin_ctzll(hit), key = page * KV4_PAGE + j;
                        const float sj = __shfl(sv, j, 64);
                        if (!A.bound.sees(key, w.last))
                            continue;
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            const int dim = 32 * d + 8 * (x >> 2) + 4 * half + (x & 3);
                            const uint32_t c = A.v_hole[ph * (KV4_PAGE * D / 2) + kv4_v_row(dim) * KV4_PAGE + j];
                            odd[x] += kKv4Parent[c >> (dim & 16 ? 4 : 0) & 15] * sj;
                        }
                    }
                }
                for (int i = f0; i < f1; ++i) {
                    const int first = s.own + (i < tiles.fsinks ? i : i + tiles.fskip) * AP_KEYS;
                    for (int key = first; key < min(first + AP_KEYS, min(wave_high + 1, s.len)); ++key) {
                        const uint16_t *from = A.v + (own_row + key) * A.v_st + h * A.v_sh + 32 * d + 4 * half;
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            const uint32_t v = from[8 * (x >> 2) + (x & 3)];
                            if ((v & 0x7F80u) == 0x7F80u && A.bound.sees(key, w.last))
                                odd[x] += __uint_as_float(v << 16);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        w.o[k][x] = k != d || odd[x] == 0.f ? w.o[k][x] : odd[x];
            }
        }
        const float l = glint_xor32(w.l, GlintAdd());
        if (take == cost) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            ap_store<D>(A.out + ((int64_t)(s.q0 + (live ? row / A.G : 0)) * A.Hq + h * A.G + (live ? row % A.G : 0)) * D, w.o, inv,
                        half, live);
        } else if (wave_live) {
            const int64_t slot = 2 * me + (at == 0); /* 1 where the group begins in this run */
            float *dst = A.part + (slot * KC_ROWS + 32 * wave + col) * D + 4 * half;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *(glint_f32x4 *)(dst + 32 * d + 2 * i) = glint_f32x4{w.o[d][i], w.o[d][i + 1], w.o[d][i + 2], w.o[d][i + 3]};
            if (half == 0)
                *(glint_f32x2 *)(A.sums + (slot * KC_ROWS + 32 * wave + col) * 2) = glint_f32x2{w.m, l};
        }
        left -= take;
        if (left == 0)
            break;
        at = 0;
        do { /* the next group that has work */
            if (++rb == A.nblk) {
                rb = 0;
                if (++h == A.H) {
                    h = 0;
                    ++b;
                }
            }
        } while (plan.pre[b * A.nblk + rb + 1] == plan.pre[b * A.nblk + rb]);
        b = __builtin_amdgcn_readfirstlane(b);
        h = __builtin_amdgcn_readfirstlane(h);
        rb = __builtin_amdgcn_readfirstlane(rb);
    }
}

/* The group that begins in workgroup w's run and ends in a later one's: its parts, added in the list's order.
 * Blocks (w, y); a block takes 32 rows, and lists are found as there. */
#define KJ_T 256
#define KJ_ROWS 32
template <int D>
__global__ __launch_bounds__(KJ_T) void k_kv4_chunk_join(KcArgs A, int grid) {
    __shared__ KcPlan plan;
    kc_plan(A, plan);
    const int total = kc_total(A, plan), share = kc_share(total, grid), me = blockIdx.x;
    const int64_t last = (int64_t)(me + 1) * share - 1; /* of the run */
    if (last >= total - 1)
        return;
    int b, h, rb, at;
    kc_find(A, plan, (int)last, b, h, rb, at);
    const int *pre = plan.pre + b * A.nblk + rb;
    const int cost = pre[1] - pre[0];
    if (at >= share || at == cost - 1) /* it began before this run, or ends with it */
        return;
    const KcSeq s = kc_seq(A, b);
    const int w_last = (int)((last + cost - 1 - at) / share);
    constexpr int LANES = D / 4;
    const int d = 4 * (threadIdx.x % LANES);
    for (int r = threadIdx.x / LANES; r < KJ_ROWS; r += KJ_T / LANES) {
        const int in = blockIdx.y * KJ_ROWS + r, row = rb * KC_ROWS + in;
        if (row >= s.rows)
            break;
        auto slot = [&](int w) { return (int64_t)(2 * w + (w == me)) * KC_ROWS + in; };
        float m = -INFINITY;
        for (int w = me; w <= w_last; ++w)
            m = fmaxf(m, A.sums[slot(w) * 2]);
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        glint_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int w = me; w <= w_last; ++w) {
            const glint_f32x2 ml = *(const glint_f32x2 *)(A.sums + slot(w) * 2);
            const glint_f32x4 v = *(const glint_f32x4 *)(A.part + slot(w) * D + d);
            const float f = __builtin_amdgcn_exp2f(ml.x - base);
            l = fmaf(f, ml.y, l);
#pragma unroll
            for (int x = 0; x < 4; ++x)
                o[x] = fmaf(f, v[x], o[x]);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *(glint_u32x2 *)(A.out + ((int64_t)(s.q0 + row / A.G) * A.Hq + h * A.G + row % A.G) * D + d) =
            glint_u32x2{glint_cvt_bf16x2(o[0] * inv, o[1] * inv), glint_cvt_bf16x2(o[2] * inv, o[3] * inv)};
    }
}

/* Sequences of a launch (0: not even one), and its workgroups. */
static int64_t kc_launch(int B, int max_q, int H, int G, int max_pages, int &nblk, int &grid) {
    nblk = (int)(((int64_t)max_q * G + KC_ROWS - 1) / KC_ROWS);
    /* units of a row block: pages, tiles of own keys, and the one of a block that sees nothing */
    const int64_t units = (int64_t)max_pages + max_q / AP_KEYS + 2;
    if (nblk > KC_PAIRS || units * nblk > (1 << 30) / H)
        return 0;
    const int64_t most = std::min<int64_t>({KC_PAIRS / nblk, (1 << 30) / (units * nblk * H), B});
    grid = (int)std::min<int64_t>(glint_cu_count(), (most * nblk * H * units + KC_SHARE - 1) / KC_SHARE);
    return most;
}
static bool kc_shape(int B, int max_q, int Hq, int H, int D, int max_pages) {
    return B >= 0 && max_q >= 1 && H >= 1 && Hq >= H && Hq % H == 0 && Hq <= 65535 && (D == 64 || D == 128) &&
           max_pages >= 1 && max_pages <= 1 << 24 && (int64_t)max_q * (Hq / H) <= (int64_t)KC_PAIRS * KC_ROWS;
}

GLINT_API int64_t glint_kv4_attend_chunk_scratch(int B, int max_q, int Hq, int H, int D, int max_pages) {
    int nblk, grid;
    if (!kc_shape(B, max_q, Hq, H, D, max_pages) || (B && !kc_launch(B, max_q, H, Hq / H, max_pages, nblk, grid)))
        return -2;
    return B ? (int64_t)grid * 2 * KC_ROWS * (D + 2) * 4 : 0;
}

GLINT_API int glint_kv4_attend_chunk(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq,
                                     const uint8_t *k_hole, const float *k_absmax, const uint8_t *v_hole,
                                     const float *v_absmax, int64_t pages, const int32_t *table, int64_t table_stride,
                                     int max_pages, const int32_t *lens, const int32_t *cu_q, int B, int max_q, int Hq, int H,
                                     int D, const uint16_t *k, int64_t k_stride_t, int64_t k_stride_h, const uint16_t *v,
                                     int64_t v_stride_t, int64_t v_stride_h, float scale, int window, int sinks,
                                     uint16_t *out, void *scratch, int64_t scratch_bytes, struct ihipStream_t *stream) {
    if (!q || !k_hole || !k_absmax || !v_hole || !v_absmax || !table || !lens || !out || !scratch || !k != !v)
        return -1;
    if (!kc_shape(B, max_q, Hq, H, D, max_pages) || Tq < 0 || Tq > INT32_MAX || pages < 1 || pages >= (int64_t)1 << 40 ||
        (!cu_q && Tq != (int64_t)B * max_q) || window < 0 || window > GLINT_WINDOW_MAX || sinks < 0)
        return -2;
    if (!glint_aligned(q, 16) || !glint_aligned(out, 16) || !glint_aligned(k_hole, 16) || !glint_aligned(v_hole, 16) ||
        !glint_aligned(k_absmax, 16) || !glint_aligned(v_absmax, 16) || !glint_aligned(scratch, 16) ||
        ((q_stride_t | q_stride_h) & 7))
        return -2;
    if (k && (!glint_aligned(k, 16) || !glint_aligned(v, 16) || ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7) ||
              k_stride_t < D || v_stride_t < D || k_stride_t > 1 << 24 || v_stride_t > 1 << 24))
        return -2;
    if (B == 0 || Tq == 0)
        return 0;
    const float scale2 = fabsf(scale) * 1.44269504088896341f;
    KcArgs a{q, q_stride_t, q_stride_h, Tq, k_hole, v_hole, k_absmax, v_absmax, pages, table, table_stride, max_pages, lens,
             cu_q, k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, B, max_q, Hq, H, Hq / H, 0,
             scale2 < FLT_MIN ? FLT_MIN : scale2, scale < 0.f ? 0x80008000u : 0u, out,
             {window ? window : GLINT_WINDOW_MAX, window ? sinks : 0}, (float *)scratch, nullptr};
    int grid;
    const int64_t most = kc_launch(B, max_q, H, a.G, max_pages, a.nblk, grid);
    if (!most || scratch_bytes < (int64_t)grid * 2 * KC_ROWS * (D + 2) * 4)
        return -2;
    a.sums = a.part + (int64_t)grid * 2 * KC_ROWS * D;
    for (int64_t b = 0; b < B; b += most) {
        a.B = (int)std::min<int64_t>(B - b, most);
        a.table = table + b * table_stride;
        a.lens = lens + b;
        if (cu_q) {
            a.cu_q = cu_q + b;
        } else { /* rows by number: this launch's alone */
            const int64_t first = b * max_q;
            a.q = q + first * q_stride_t;
            a.out = out + first * Hq * D;
            a.Tq = (int64_t)a.B * max_q;
            if (k) {
                a.k = k + first * k_stride_t;
                a.v = v + first * v_stride_t;
            }
        }
        const dim3 join(grid, KC_ROWS / KJ_ROWS);
        if (D == 64) {
            k_kv4_chunk<64><<<grid, KC_T, 0, stream>>>(a);
            k_kv4_chunk_join<64><<<join, KJ_T, 0, stream>>>(a, grid);
        } else {
            k_kv4_chunk<128><<<grid, KC_T, 0, stream>>>(a);
            k_kv4_chunk_join<128><<<join, KJ_T, 0, stream>>>(a, grid);
        }
        if (hipGetLastError() != hipSuccess)
            return -3;
    }
    return 0;
}
