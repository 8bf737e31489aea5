/* Attention of chunks of new tokens over the 4-bit cache (include/glint_serve.h), in three launches.
 *
 * k_kv4_unpack — every tile of 64 keys and values that a sequence's rows see, once per key head: cached
 *   pages' codes, and, where the call brings them, the new tokens' own BF16 rows, become f16 operands in
 *   scratch memory, K as [64][D] and V^T as [D][64], in the very order in which the next kernel's LDS holds
 *   them. A tile is scaled by a power of two, so that f16 keeps 11 bits of PARENT * absmax (one rounding) and
 *   all bits of a BF16 element. Decoding in the attention kernel itself, once for 256 query rows, took 586 us
 *   for 2048 tokens over 16384 where this takes X: its LDS round trips lie in every wave's way, and a
 *   document's chunk has many row blocks.
 *
 * k_kv4_chunk — a group is one sequence, key head and block of up to 128 query rows (the heads that share the
 *   key head, times the new tokens), its work the tiles that its rows see. The groups' tiles form one list, and
 *   every workgroup takes an equal run of it, so that a long context under few rows fills the device and a
 *   ragged batch is shared out evenly. Per tile it is glint_attend_prompt.hip's kernel in f16: S^T = K Q^T, the
 *   weights feed O^T = V^T P^T as they lie; V^T's tokens lie in that order, so both operands are plain 16-B
 *   reads. Tiles come by the loads' direct path to LDS, one ahead.
 *
 * k_kv4_chunk_join — parts of a group that lies in several runs, added in the list's order.
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

#define KC_WAVES 4
#define KC_T (64 * KC_WAVES)
#define KC_ROWS (32 * KC_WAVES)
#define KC_PAIRS 2048 /* of a sequence and a row block, in a launch */
#define KC_SHARE 2    /* tiles that a workgroup takes at least */
#define KC_UP 7.f     /* weights are 2^KC_UP times the softmax's: f16 has room above, and its small ones keep more bits */
#define KC_CAP ((int64_t)1 << 31) /* bytes of tiles of a launch */

/* What a tile's elements were multiplied by. */
struct KcMeta {
    float kback;   /* the inverse of the keys' power */
    uint32_t vexp; /* the values': 2^(14 - e), e + KC_EXP here; and */
};
#define KC_EXP 1024
#define KC_ABSENT 0x80000000u /* the page is not in the pool: nothing was written */
#define KC_ODD 0x40000000u    /* a value that is not finite was taken out */

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
    int h0, Hn;   /* key heads of this launch */
    int slots;    /* tiles of a sequence and head: max_pages, then own keys' */
    float scale2; /* |scale| log2 e, above 0 */
    uint32_t q_sign; /* 0x80008000 where the scale is negative */
    uint16_t *out;
    ApBound bound;
    float *part; /* outputs of two parts per workgroup, [KC_ROWS][D] each, */
    float *sums; /* and their rows' maxima and sums */
    KcMeta *meta;
    char *tiles;
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
/* The tiles that row blocks rb .. rb + blocks - 1 see: step i of the first np is page i, or, past the sinks', i + pskip; then nf tiles of own
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
__device__ __forceinline__ KcTiles kc_tiles(const KcArgs &a, const KcSeq &s, int rb, int blocks) {
    KcTiles t{0, 0, 0, 0, 0, 0};
    if (rb * KC_ROWS >= s.rows)
        return t;
    const int p0 = s.len - s.nq + rb * KC_ROWS / a.G;
    const int p1 = s.len - s.nq + min(s.rows - 1, (rb + blocks) * KC_ROWS - 1) / a.G;
    const int64_t low = (int64_t)p0 - a.bound.window + 1;
    kc_range(min(s.held - 1, p1), low, a.bound.sinks, t.np, t.psinks, t.pskip);
    if (a.k)
        kc_range(p1 - s.own, low - s.own, (int64_t)a.bound.sinks - s.own, t.nf, t.fsinks, t.fskip);
    return t;
}
/* A row block that sees nothing counts as one tile: its rows are zero. */
__device__ __forceinline__ int kc_cost(const KcArgs &a, const KcSeq &s, int rb) {
    const KcTiles t = kc_tiles(a, s, rb, 1);
    return rb * KC_ROWS < s.rows ? max(1, t.np + t.nf) : 0;
}

/* The list: sequences, of each its key heads, of each its row blocks. pre[i] is the cost of the pairs
 * (sequence, row block) before pair i. */
struct KcPlan {
    int pre[KC_PAIRS + 1];
    int wave[KC_WAVES];
    int b, rb, at;
};
template <class F> /* pairs, and the cost of pair i */
__device__ __forceinline__ void kc_scan(KcPlan &p, int pairs, F cost_of) {
    const int threads = blockDim.x, per = (pairs + threads - 1) / threads, lane = threadIdx.x & 63;
#pragma unroll 1
    for (int i = threadIdx.x; i < pairs; i += threads)
        p.pre[i] = cost_of(i);
    __syncthreads();
    const int first = min((int)threadIdx.x * per, pairs), end = min(first + per, pairs);
    int sum = 0;
#pragma unroll 1
    for (int i = first; i < end; ++i)
        sum += p.pre[i];
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
#pragma unroll 1
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w)
        before += p.wave[w];
#pragma unroll 1
    for (int i = first; i < end; ++i) {
        const int cost = p.pre[i];
        p.pre[i] = before;
        before += cost;
    }
    if (end == pairs && first < pairs)
        p.pre[pairs] = before;
    __syncthreads();
}
__device__ __forceinline__ void kc_plan(const KcArgs &a, KcPlan &p) {
    kc_scan(p, a.B * a.nblk, [&](int i) { return kc_cost(a, kc_seq(a, i / a.nblk), i % a.nblk); });
}
/* The group that unit u of the list lies in, and where in it. */
__device__ __forceinline__ void kc_find(const KcArgs &a, KcPlan &p, int u, int &b, int &h, int &rb, int &at) {
    for (int i = threadIdx.x; i < a.B; i += blockDim.x)
        if (a.Hn * p.pre[i * a.nblk] <= u && u < a.Hn * p.pre[(i + 1) * a.nblk])
            p.b = i;
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(p.b);
    const int *pre = p.pre + b * a.nblk;
    const int each = pre[a.nblk] - pre[0], in = u - a.Hn * pre[0];
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
    return __builtin_amdgcn_readfirstlane(a.Hn * p.pre[a.B * a.nblk]);
}
__device__ __forceinline__ int kc_share(int total, int grid) { return max(KC_SHARE, (total + grid - 1) / grid); }

union KcFrag {
    uint32_t u[4];
    glint_u32x4 v;
    kc_f16x8 f;
};
__device__ __forceinline__ uint32_t kc_f16pair(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(glint_f32x2{lo, hi}, kc_f16x2));
}
/* The place of tile `at` (a page, or past max_pages own keys) of sequence b and head h of the launch. */
__device__ __forceinline__ int64_t kc_slot(const KcArgs &a, int b, int h, int at) { return ((int64_t)b * a.Hn + h) * a.slots + at; }
/* Where V^T's 16-B chunk c of dimension d lies in a row of 128 B: 16 lanes reading one chunk of 16 rows touch every
 * bank once. Chunk 2 g + y holds tokens 16 g + 4 y + 0..3 and 8 on. */
__device__ __forceinline__ int kc_v_at(int d, int c) { return d * 128 + 16 * (c ^ ((d >> 1) & 7)); }

/* ------------------------------------------------------------------ tiles */
#define KU_T 256
#define KU_COPIES 16 /* of an entry, 8 B each */

/* The exponent e of a power of two 2^(14 - e) that brings `top` (finite) under 2^15, in steps of `step`. */
__device__ __forceinline__ int ku_exponent(float top, int step) {
    const int e = max(-112, (int)(__float_as_uint(top) >> 23) - 127);
    return (e + step - 1) & -step;
}

template <int D>
__global__ __launch_bounds__(KU_T) void k_kv4_unpack(KcArgs A) {
    constexpr int NB = D / 64, TILE = AP_KEYS * D * 2, CH = D / 8;
    __shared__ __attribute__((aligned(16))) glint_f32x2 entries[256 * KU_COPIES]; /* a byte's two parents */
    __shared__ __attribute__((aligned(16))) uint16_t rows[AP_KEYS][D + 2];        /* own values, to be turned */
    __shared__ float tops[2][KU_T / 64];
    __shared__ uint32_t odds;
    __shared__ KcPlan plan;
    for (int i = threadIdx.x; i < 256 * KU_COPIES; i += KU_T)
        entries[i] = glint_f32x2{kKv4Parent[i / KU_COPIES & 15], kKv4Parent[i / KU_COPIES >> 4]};
    /* the list: a sequence's tiles, head after head */
    kc_scan(plan, A.B, [&](int b) {
        const KcTiles t = kc_tiles(A, kc_seq(A, b), 0, A.nblk);
        return t.np + t.nf;
    });
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int total = A.Hn * plan.pre[A.B];
    int b = 0;
    for (int u = blockIdx.x; u < total; u += gridDim.x) {
        while (A.Hn * plan.pre[b + 1] <= u) /* u only grows */
            ++b;
        b = __builtin_amdgcn_readfirstlane(b);
        const int each = plan.pre[b + 1] - plan.pre[b], in = u - A.Hn * plan.pre[b];
        const int hl = in / each, i = in % each, h = A.h0 + hl;
        const KcSeq s = kc_seq(A, b);
        const KcTiles t = kc_tiles(A, s, 0, A.nblk);
        const int gap = s.len - s.nq;
        const int low = gap - A.bound.window + 1, high = gap + (s.rows - 1) / A.G; /* what some row sees */
        auto seen = [&](int key) { return key <= high && (key >= low || key < A.bound.sinks); };
        KcMeta meta{1.f, KC_EXP};
        if (i < t.np) {
            const int page = i < t.psinks ? i : i + t.pskip, key = page * KV4_PAGE;
            const int64_t slot = kc_slot(A, b, hl, page);
            char *kt = A.tiles + slot * (2 * TILE), *vt = kt + TILE;
            const int pid = A.table[(int64_t)b * A.table_stride + page];
            if (pid < 0 || pid >= A.pages) {
                if (threadIdx.x == 0)
                    A.meta[slot] = KcMeta{1.f, KC_ABSENT};
                continue;
            }
            const int64_t ph = (int64_t)pid * A.H + h;
            const float *ka = A.k_absmax + ph * (NB * KV4_PAGE), *va = A.v_absmax + ph * (NB * KV4_PAGE);
            const bool mine = key + lane < s.held && seen(key + lane);
            /* a thread's codes: NB times 8 B of a key row (dimensions 64 x + 16 part ..), 16 B of a value row */
            const int tok = threadIdx.x >> 2, part = threadIdx.x & 3;
            const uint8_t *kp = A.k_hole + (ph * KV4_PAGE + tok) * (D / 2) + part * (8 * NB);
            const uint8_t *vp = A.v_hole + (ph * (D / 2) + tok) * KV4_PAGE + 16 * part; /* row tok, group part */
            const bool has_v = tok < D / 2;
            uint32_t kw[NB][2], vw[4];
            float ks[NB], kl[NB], vl[NB];
            glint_f32x4 vs[4];
            const int dim = ((tok >> 4) << 5) + (tok & 15); /* of the low nibbles; the high ones' is 16 on */
#pragma unroll
            for (int x = 0; x < NB; ++x) {
                kw[x][0] = ((const uint32_t *)kp)[2 * x];
                kw[x][1] = ((const uint32_t *)kp)[2 * x + 1];
                ks[x] = ka[x * KV4_PAGE + tok];
                kl[x] = ka[x * KV4_PAGE + lane];
                vl[x] = va[x * KV4_PAGE + lane];
            }
            if (has_v) {
                const glint_u32x4 w = *(const glint_u32x4 *)vp;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    vw[j] = w[j];
                    vs[j] = *(const glint_f32x4 *)(va + (dim >> 6) * KV4_PAGE + 16 * part + 4 * j);
                }
            }
            float ktop = 0.f, vtop = 0.f;
            bool odd = false;
#pragma unroll
            for (int x = 0; x < NB; ++x) {
                ktop = fabsf(kl[x]) <= FLT_MAX ? fmaxf(ktop, fabsf(kl[x])) : ktop;
                vtop = fabsf(vl[x]) <= FLT_MAX ? fmaxf(vtop, fabsf(vl[x])) : vtop;
                odd |= !(fabsf(vl[x]) <= FLT_MAX);
            }
            const int ke = ku_exponent(glint_wave_max(mine ? ktop : 0.f), 1), ve = ku_exponent(glint_wave_max(mine ? vtop : 0.f), 8);
            const float kdown = ldexpf(1.f, 14 - ke), vdown = ldexpf(1.f, 14 - ve);
            meta = KcMeta{ldexpf(1.f, ke - 14), (uint32_t)(ve + KC_EXP) | (__any(mine && odd) ? KC_ODD : 0u)};
            if (threadIdx.x == 0)
                A.meta[slot] = meta;
            const glint_f32x2 *entry = entries + (lane & (KU_COPIES - 1));
            auto pair = [&](uint32_t word, int byte) { return entry[(word >> (8 * byte) & 255u) * KU_COPIES]; };
#pragma unroll
            for (int x = 0; x < NB; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    glint_u32x4 eight;
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const glint_f32x2 e = pair(kw[x][y], z);
                        eight[z] = kc_f16pair(e.x * (ks[x] * kdown), e.y * (ks[x] * kdown));
                    }
                    *(glint_u32x4 *)(kt + tok * (D * 2) + 16 * ap_k_chunk<D>(tok, 8 * x + 2 * part + y)) = eight;
                }
            if (has_v) {
#pragma unroll
                for (int y = 0; y < 2; ++y) { /* chunk 2 part + y: words y and y + 2 */
                    glint_u32x4 lo, hi;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int j = y + 2 * x;
                        float a[4], z[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int at = key + 16 * part + 4 * j + k;
                            /* what nobody sees is 0: a weight of 0 does not undo an infinity */
                            const float f = fabsf(vs[j][k]) <= FLT_MAX && at < s.held && seen(at) ? vs[j][k] * vdown : 0.f;
                            const glint_f32x2 e = pair(vw[j], k);
                            a[k] = e.x * f;
                            z[k] = e.y * f;
                        }
                        lo[2 * x] = kc_f16pair(a[0], a[1]);
                        lo[2 * x + 1] = kc_f16pair(a[2], a[3]);
                        hi[2 * x] = kc_f16pair(z[0], z[1]);
                        hi[2 * x + 1] = kc_f16pair(z[2], z[3]);
                    }
                    *(glint_u32x4 *)(vt + kc_v_at(dim, 2 * part + y)) = lo;
                    *(glint_u32x4 *)(vt + kc_v_at(dim + 16, 2 * part + y)) = hi;
                }
            }
        } else {
            /* own keys: positions s.own + 64 f ..; rows past the sequence's last are 0 */
            const int f = i - t.np < t.fsinks ? i - t.np : i - t.np + t.fskip;
            const int64_t slot = kc_slot(A, b, hl, A.max_pages + f);
            char *kt = A.tiles + slot * (2 * TILE), *vt = kt + TILE;
            const int key = s.own + f * AP_KEYS;
            const int64_t row0 = (int64_t)s.q0 + s.nq - s.len + key;
            constexpr int PER = AP_KEYS * CH / KU_T; /* 16-B chunks of a thread */
            glint_u32x4 kx[PER], vx[PER];
            float ktop = 0.f, vtop = 0.f;
            bool odd = false;
            __syncthreads(); /* the tile before has been turned, odds and tops are read */
            if (threadIdx.x == 0)
                odds = 0;
#pragma unroll
            for (int x = 0; x < PER; ++x) {
                const int r = (threadIdx.x + x * KU_T) / CH, c = (threadIdx.x + x * KU_T) % CH;
                const bool mine = key + r < s.len && seen(key + r);
                kx[x] = vx[x] = glint_u32x4{0, 0, 0, 0};
                if (mine) {
                    kx[x] = *(const glint_u32x4 *)(A.k + (row0 + r) * A.k_st + h * A.k_sh + 8 * c);
                    vx[x] = *(const glint_u32x4 *)(A.v + (row0 + r) * A.v_st + h * A.v_sh + 8 * c);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float a = fabsf(k ? glint_bf16hi(kx[x][j]) : glint_bf16lo(kx[x][j]));
                        const float z = fabsf(k ? glint_bf16hi(vx[x][j]) : glint_bf16lo(vx[x][j]));
                        ktop = a <= FLT_MAX ? fmaxf(ktop, a) : ktop;
                        if (z <= FLT_MAX) {
                            vtop = fmaxf(vtop, z);
                        } else {
                            odd = true;
                            vx[x][j] &= k ? 0xFFFFu : 0xFFFF0000u;
                        }
                    }
            }
            ktop = glint_wave_max(ktop);
            vtop = glint_wave_max(vtop);
            if (lane == 0) {
                tops[0][wave] = ktop;
                tops[1][wave] = vtop;
            }
            __syncthreads();
            if (odd)
                odds = 1;
#pragma unroll
            for (int x = 0; x < KU_T / 64; ++x) {
                ktop = fmaxf(ktop, tops[0][x]);
                vtop = fmaxf(vtop, tops[1][x]);
            }
            const int ke = ku_exponent(ktop, 1), ve = ku_exponent(vtop, 8);
            const float kdown = ldexpf(1.f, 14 - ke), vdown = ldexpf(1.f, 14 - ve);
#pragma unroll
            for (int x = 0; x < PER; ++x) {
                const int r = (threadIdx.x + x * KU_T) / CH, c = (threadIdx.x + x * KU_T) % CH;
                glint_u32x4 eight;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    eight[j] = kc_f16pair(glint_bf16lo(kx[x][j]) * kdown, glint_bf16hi(kx[x][j]) * kdown);
                    const uint32_t two = kc_f16pair(glint_bf16lo(vx[x][j]) * vdown, glint_bf16hi(vx[x][j]) * vdown);
                    *(uint32_t *)&rows[r][8 * c + 2 * j] = two;
                }
                *(glint_u32x4 *)(kt + r * (D * 2) + 16 * ap_k_chunk<D>(r, c)) = eight;
            }
            __syncthreads();
            if (threadIdx.x == 0)
                A.meta[slot] = KcMeta{ldexpf(1.f, ke - 14), (uint32_t)(ve + KC_EXP) | (odds ? KC_ODD : 0u)};
#pragma unroll
            for (int x = 0; x < PER; ++x) {
                const int d = (threadIdx.x + x * KU_T) / 8, c = (threadIdx.x + x * KU_T) % 8;
                const int first = 16 * (c >> 1) + 4 * (c & 1);
                glint_u32x4 eight;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = first + (j & 1) * 2 + (j >> 1) * 8;
                    eight[j] = rows[r][d] | (uint32_t)rows[r + 1][d] << 16;
                }
                *(glint_u32x4 *)(vt + kc_v_at(d, c)) = eight;
            }
        }
    }
}

/* ------------------------------------------------------------------ attention */
/* A page's scores: as ap_tile's, in f16. Products in groups of four: the next group's operands are read ahead of a
 * group's products, whose time covers the reads' latency; left to itself the compiler waits for every read. */
typedef const __attribute__((address_space(3))) glint_u32x4 kc_lds_u32x4;
template <int D>
__device__ __forceinline__ void kc_scores(const ap_lds *kl, const ApRows<D> &w, ap_f32x16 (&sc)[2]) {
    KcFrag f[2][4];
    auto read = [&](int g) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int s = 2 * g + (x >> 1), a = x & 1;
            f[g & 1][x].v = *(kc_lds_u32x4 *)(kl + (w.kat[s & 3] ^ (128 * (s >> 2))) + a * 32 * D * 2);
        }
    };
    read(0);
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sc[a][i] = 0.f;
#pragma unroll
    for (int g = 0; g < D / 32; ++g) {
        if (g + 1 < D / 32)
            read(g + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            KcFrag q;
            q.v = w.q[2 * g + (x >> 1)].v;
            sc[x & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[g & 1][x].f, q.f, sc[x & 1], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}
/* What the scores weigh: `upto` is the last key of the tile that the lane's row may see. Values are V^T; the weights are
 * multiplied by `less`, a power of two, where it is not 1. */
template <int D>
__device__ __forceinline__ void kc_weigh(const ap_lds *vl, int at, ApRows<D> &w, ap_f32x16 (&sc)[2], const uint32_t (&vat)[4],
                                         float factor, float less, bool masked, int upto, int half, const ApBound &bound) {
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
    constexpr int PARTS = D / 32; /* of the outputs */
    KcFrag f[2][4];
    auto read = [&](int g) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
            f[g & 1][x].v = *(kc_lds_u32x4 *)(vl + vat[(4 * g + x) / PARTS] + (4 * g + x) % PARTS * 32 * 128);
    };
    read(0);
    __builtin_amdgcn_sched_barrier(0);
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
    if (less != 1.f) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
            pf[s].f *= (_Float16)less;
    }
#pragma unroll
    for (int g = 0; g < PARTS; ++g) {
        if (g + 1 < PARTS)
            read(g + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int s = (4 * g + x) / PARTS, d = (4 * g + x) % PARTS;
            w.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[g & 1][x].f, pf[s].f, w.o[d], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <int D>
__global__ __launch_bounds__(KC_T, 2) void k_kv4_chunk(KcArgs A) {
    constexpr int TILE = AP_KEYS * D * 2, LOADS = TILE / (16 * KC_T);
    /* arrays of their own, so that reads of one do not wait for loads into the other */
    __shared__ __attribute__((aligned(16))) char k0t[TILE], k1t[TILE], v0t[TILE], v1t[TILE];
    __shared__ KcPlan plan;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    kc_plan(A, plan);
    const int grid = gridDim.x, total = kc_total(A, plan), share = kc_share(total, grid);
    /* neighbours in the list share keys: they go to one XCD, a workgroup's being its index modulo 8 */
    const int me = grid & 7 ? (int)blockIdx.x : ((int)blockIdx.x & 7) * (grid >> 3) + ((int)blockIdx.x >> 3);
    if ((int64_t)me * share >= total)
        return;
    int left = min(share, total - me * share); /* of this workgroup's run */
    int b, h, rb, at;
    kc_find(A, plan, me * share, b, h, rb, at);

    ApRows<D> w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w.kat[j] = col * D * 2 + 16 * ap_k_chunk<D>(col, 2 * j + half);
    uint32_t vat[4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
        vat[s] = kc_v_at(col, 2 * s + half);

    for (;;) {
        const KcSeq s = kc_seq(A, b);
        const KcTiles tiles = kc_tiles(A, s, rb, 1);
        const int n = tiles.np + tiles.nf, cost = max(1, n);
        const int take = min(left, cost - at), end = min(at + take, n); /* tiles at .. end - 1 */
        const int row = rb * KC_ROWS + 32 * wave + col, head = (A.h0 + h) * A.G;
        const bool live = row < s.rows, wave_live = rb * KC_ROWS + 32 * wave < s.rows;
        const int gap = s.len - s.nq;
        const int wave_low = gap + (rb * KC_ROWS + 32 * wave) / A.G;
        const int wave_high = gap + min(s.rows - 1, rb * KC_ROWS + 32 * wave + 31) / A.G;
        w.m = -INFINITY;
        w.l = 0.f;
        w.last = live ? gap + row / A.G : -1;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                w.o[d][i] = 0.f;
        bool apart = false;
        int oexp = -4096; /* the outputs are 2^(14 - oexp) times themselves */
        if (at < end) {
            /* the place of tile i: pages, then own keys; its first position and, of what it holds, the end */
            auto place = [&](int i) {
                return i < tiles.np ? (i < tiles.psinks ? i : i + tiles.pskip)
                                    : A.max_pages + (i - tiles.np < tiles.fsinks ? i - tiles.np : i - tiles.np + tiles.fskip);
            };
            const int64_t slot0 = kc_slot(A, b, h, 0);
            const uint32_t my = threadIdx.x * 16;
            auto fetch = [&](int i, ap_lds *kt, ap_lds *vt) {
                const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                    (void *)(A.tiles + (slot0 + place(i)) * (2 * TILE)), (short)0, 2 * TILE, GLINT_BUF_DWORD3);
#pragma unroll
                for (int x = 0; x < LOADS; ++x)
                    ap_dma(r, kt + (x * KC_T + wave * 64) * 16, my, x * (KC_T * 16));
#pragma unroll
                for (int x = 0; x < LOADS; ++x)
                    ap_dma(r, vt + (x * KC_T + wave * 64) * 16, my, TILE + x * (KC_T * 16));
            };
            __syncthreads(); /* the last group's tiles are read */
            fetch(at, (ap_lds *)k0t, (ap_lds *)v0t);
            /* q as f16, scaled to 2^14 .. 2^15 by a power of two of the row's */
            const uint16_t *qr = A.q + (int64_t)(s.q0 + (live ? row / A.G : 0)) * A.q_st + (head + (live ? row % A.G : 0)) * A.q_sh;
            uint32_t high = 0;
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
                w.q[x].v = *(const glint_u32x4 *)(qr + 16 * x + 8 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w.q[x].u[i] ^= A.q_sign;
                    high = max(high, max((w.q[x].u[i] & 0x7FFFu) << 16, w.q[x].u[i] & 0x7FFF0000u));
                }
            }
            high = __float_as_uint(glint_xor32(__uint_as_float(min(high, 0x7F800000u)), GlintMax()));
            const int ex = high >= 0x7F800000u ? 0 : (int)(high >> 23) - 127 - 14;
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w.q[x].u[i] = kc_f16pair(ldexpf(glint_bf16lo(w.q[x].u[i]), -ex), ldexpf(glint_bf16hi(w.q[x].u[i]), -ex));
            const float factor = ldexpf(A.scale2, ex);

            auto step = [&](int i, ap_lds *kt, ap_lds *vt, ap_lds *kn, ap_lds *vn) {
                const int to = place(i);
                const bool own = i >= tiles.np;
                const int key = own ? s.own + (to - A.max_pages) * AP_KEYS : to * AP_KEYS;
                const int ends = own ? INT32_MAX : s.held - 1; /* the last position that the tile may show */
                const KcMeta meta = A.meta[slot0 + to];
                __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0); /* this wave's part of the tile */
                __syncthreads();
                if (i + 1 < end)
                    fetch(i + 1, kn, vn); /* over the tile before, which every wave has left */
                apart |= (meta.vexp & KC_ODD) != 0;
                if ((meta.vexp & KC_ABSENT) || !wave_live || key > min(wave_high, ends) ||
                    !(key + AP_KEYS - 1 > wave_low - A.bound.window || key < A.bound.sinks))
                    return;
                ap_f32x16 sc[2];
                kc_scores<D>(kt, w, sc);
                const int ve = (int)(meta.vexp & 0xFFFFu) - KC_EXP;
                if (ve > oexp) {
                    const float by = ldexpf(1.f, max(oexp - ve, -300));
#pragma unroll
                    for (int d = 0; d < D / 32; ++d)
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            w.o[d][x] *= by;
                    oexp = ve;
                }
                const bool all = key > wave_high - A.bound.window || key + AP_KEYS <= A.bound.sinks;
                kc_weigh<D>(vt, key, w, sc, vat, fminf(fmaxf(factor * meta.kback, FLT_MIN), FLT_MAX), ldexpf(1.f, max(ve - oexp, -30)),
                            key + AP_KEYS - 1 > min(wave_low, ends) || !all, min(w.last, ends), half, A.bound);
            };
            for (int i = at; i < end; i += 2) {
                step(i, (ap_lds *)k0t, (ap_lds *)v0t, (ap_lds *)k1t, (ap_lds *)v1t);
                if (i + 1 < end)
                    step(i + 1, (ap_lds *)k1t, (ap_lds *)v1t, (ap_lds *)k0t, (ap_lds *)v0t);
            }
            const float back = ldexpf(1.f, max(oexp - 14, -300));
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    w.o[d][x] *= back;
        }

        /* A value that is not finite leaves itself or NaN in its dimension of the rows that see it, whatever its
         * weight. */
        if (apart) {
#pragma unroll 1
            for (int d = 0; d < D / 32; ++d) {
                ap_f32x16 odd;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    odd[i] = 0.f;
                for (int i = at; i < min(end, tiles.np); ++i) {
                    const int page = i < tiles.psinks ? i : i + tiles.pskip;
                    const int pid = A.table[(int64_t)b * A.table_stride + page];
                    if (pid < 0 || pid >= A.pages)
                        continue;
                    const int64_t ph = (int64_t)pid * A.H + A.h0 + h;
                    const float sv = A.v_absmax[ph * (D / 64 * KV4_PAGE) + (d >> 1) * KV4_PAGE + lane];
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
                for (int i = max(at, tiles.np); i < end; ++i) {
                    const int f = i - tiles.np < tiles.fsinks ? i - tiles.np : i - tiles.np + tiles.fskip;
                    const int first = s.own + f * AP_KEYS;
                    for (int key = first; key < min(first + AP_KEYS, min(wave_high + 1, s.len)); ++key) {
                        const uint16_t *from = A.v + ((int64_t)s.q0 + s.nq - s.len + key) * A.v_st + (A.h0 + h) * A.v_sh + 32 * d + 4 * half;
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
            ap_store<D>(A.out + ((int64_t)(s.q0 + (live ? row / A.G : 0)) * A.Hq + head + (live ? row % A.G : 0)) * D, w.o, inv,
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
                if (++h == A.Hn) {
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
        *(glint_u32x2 *)(A.out + ((int64_t)(s.q0 + row / A.G) * A.Hq + (A.h0 + h) * A.G + row % A.G) * D + d) =
            glint_u32x2{glint_cvt_bf16x2(o[0] * inv, o[1] * inv), glint_cvt_bf16x2(o[2] * inv, o[3] * inv)};
    }
}

/* How a call is cut into launches: sequences and key heads of one, its tiles a sequence and head, workgroups; and the
 * scratch memory's parts. No sequence fits: seqs is 0. */
struct KcCut {
    int64_t seqs;
    int heads, slots, nblk, grid;
    int64_t sums, meta, tiles, bytes; /* offsets; all of it */
};
static KcCut kc_cut(int B, int max_q, int H, int G, int D, int max_pages, bool own) {
    KcCut c{};
    c.nblk = (int)(((int64_t)max_q * G + KC_ROWS - 1) / KC_ROWS);
    c.slots = max_pages + (own ? max_q / AP_KEYS + 1 : 0);
    const int64_t tile = (int64_t)4 * AP_KEYS * D * c.slots; /* bytes of a sequence and head */
    const int64_t units = (int64_t)c.slots + 1;              /* of a row block; one that sees nothing counts as 1 */
    if (c.nblk > KC_PAIRS || units * c.nblk > (1 << 30) / H)
        return c;
    c.heads = (int)std::max<int64_t>(1, std::min<int64_t>(H, KC_CAP / tile));
    c.seqs = std::min<int64_t>({KC_PAIRS / c.nblk, (1 << 30) / (units * c.nblk * H), B});
    c.seqs = std::max<int64_t>(1, std::min<int64_t>(c.seqs, KC_CAP / (tile * c.heads)));
    c.grid = (int)std::min<int64_t>(2 * glint_cu_count(), (c.seqs * c.nblk * c.heads * units + KC_SHARE - 1) / KC_SHARE);
    c.sums = (int64_t)c.grid * 2 * KC_ROWS * D * 4;
    c.meta = c.sums + (int64_t)c.grid * 2 * KC_ROWS * 2 * 4;
    const int64_t slots = c.seqs * c.heads * c.slots;
    c.tiles = (c.meta + slots * (int64_t)sizeof(KcMeta) + 255) & -256;
    c.bytes = c.tiles + slots * 4 * AP_KEYS * D;
    return c;
}
static bool kc_shape(int B, int max_q, int Hq, int H, int D, int max_pages) {
    return B >= 0 && max_q >= 1 && H >= 1 && Hq >= H && Hq % H == 0 && Hq <= 65535 && (D == 64 || D == 128) &&
           max_pages >= 1 && max_pages <= 1 << 24 && (int64_t)max_q * (Hq / H) <= (int64_t)KC_PAIRS * KC_ROWS;
}

GLINT_API int64_t glint_kv4_attend_chunk_scratch(int B, int max_q, int Hq, int H, int D, int max_pages, int own) {
    if (!kc_shape(B, max_q, Hq, H, D, max_pages))
        return -2;
    if (B == 0)
        return 0;
    const KcCut c = kc_cut(B, max_q, H, Hq / H, D, max_pages, own != 0);
    return c.seqs ? c.bytes : -2;
}

template <int D>
static void kc_run(const KcArgs &a, int grid, hipStream_t stream) {
    k_kv4_unpack<D><<<grid, KU_T, 0, stream>>>(a);
    k_kv4_chunk<D><<<grid, KC_T, 0, stream>>>(a);
    k_kv4_chunk_join<D><<<dim3(grid, KC_ROWS / KJ_ROWS), KJ_T, 0, stream>>>(a, grid);
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
    const KcCut c = kc_cut(B, max_q, H, Hq / H, D, max_pages, k != nullptr);
    if (!c.seqs || scratch_bytes < c.bytes)
        return -2;
    char *const mem = (char *)scratch;
    KcArgs a{q, q_stride_t, q_stride_h, Tq, k_hole, v_hole, k_absmax, v_absmax, pages, table, table_stride, max_pages, lens,
             cu_q, k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, B, max_q, Hq, H, Hq / H, c.nblk, 0, 0, c.slots,
             scale2 < FLT_MIN ? FLT_MIN : scale2, scale < 0.f ? 0x80008000u : 0u, out,
             {window ? window : GLINT_WINDOW_MAX, window ? sinks : 0}, (float *)mem, (float *)(mem + c.sums),
             (KcMeta *)(mem + c.meta), mem + c.tiles};
    for (int64_t b = 0; b < B; b += c.seqs) {
        a.B = (int)std::min<int64_t>(B - b, c.seqs);
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
        for (a.h0 = 0; a.h0 < H; a.h0 += c.heads) {
            a.Hn = std::min(c.heads, H - a.h0);
            if (D == 64)
                kc_run<64>(a, c.grid, stream);
            else
                kc_run<128>(a, c.grid, stream);
            if (hipGetLastError() != hipSuccess)
                return -3;
        }
    }
    return 0;
}
