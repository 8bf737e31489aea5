/* Attention of chunks of new tokens over the 4-bit cache (include/glint_serve.h), in three launches.
 *
 * k_kv4_unpack — every tile of 64 keys and values that a sequence's rows see, once per key head: cached
 *   pages' codes, and, where the call brings them, the new tokens' own BF16 rows, become f16 operands in
 *   scratch memory, K as [64][D] and V^T as [D][64], in the very order in which the next kernel's LDS holds
 *   them. A tile is scaled by a power of two, so that f16 keeps 11 bits of PARENT * absmax (one rounding) and
 *   all bits of a BF16 element; what one power does not hold is marked (KC_WIDE) and taken as pairs of BF16.
 *   Decoding in the attention kernel itself, once for 256 query rows, took 586 us for 2048 tokens over 16384
 *   where this took 528: its LDS round trips lie in every wave's way, and a document's chunk has many row blocks.
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
 *   them, and LDS, from which each wave reads every tile. 2048 tokens of 32 heads of 128 over 8 after 14336: 515
 *   GFLOP in 531 to 581 us by device, of which unpacking takes 23 (its writes; 15 without them), the join 4 and
 *   the rest 0.97 PFLOP/s at some 2.0 GHz, where an 8192^3 product of the library reaches 1.2 to 1.3. 512 tokens
 *   in 4 parts a row block with their own BF16 keys: 190 to 201 us, 34 of them unpacking (where the form for own
 *   keys spills 18 registers) and 17 the join; with a window of 1024 57 to 60. */
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attend_tile.h"
#include "kv4_tile.h"

typedef _Float16 kc_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 kc_f16x2 __attribute__((ext_vector_type(2)));

#define KC_WAVES 4
#define KC_T (64 * KC_WAVES)
#define KC_ROWS (32 * KC_WAVES)
#define KC_PAIRS 2048 /* of a sequence and a row block, in a launch */
#define KC_SHARE 4    /* tiles that a workgroup takes at least */
#define KC_UP 7.f     /* weights are 2^KC_UP times the softmax's: f16 has room above, and its small ones keep more bits */
#define KC_CAP ((int64_t)1 << 31) /* bytes of tiles of a launch */
#define KC_LENGTH (INT32_MAX - AP_KEYS) /* tokens of a sequence: a tile's last position is an int wherever it begins */

/* What a tile's elements were multiplied by. */
struct KcMeta {
    float kback;   /* the inverse of the keys' power */
    uint32_t vexp; /* the values': 2^(14 - e), e + KC_EXP here; and */
};
#define KC_EXP 1024
/* What one power a tile does not keep in f16, or an output in f32 while it goes from tile to tile, makes a tile wide:
 * it is left out of these products and taken by kc_wide_tile. The size of a key or value then costs the rows nothing that do not
 * see it or give it no weight.
 *   Keys: f16 is off by 2^-25 of what an element is scaled to, q's likewise, and a score by 2^-9 D times its factor at most. A
 *   factor of KC_KEYS leaves 2^-18; a wave's rows have powers of their own, so a wave asks for itself.
 *   Values: a token's 64 dimensions whose largest is KC_SPAN of the tile's, which is 2^7 to 2^15 once scaled, keep 2^-20 of that.
 *   Powers past KC_BAND either way: tiles within are 2^64 apart at most, by which an output may be lifted. */
#define KC_KEYS 0x1p-16f
#define KC_SPAN 0x1p-12f
#define KC_BAND 32
#define KC_ABSENT 0x80000000u /* the page is not in the pool: nothing was written */
#define KC_ODD 0x40000000u    /* a value that is not finite was taken out */
#define KC_WIDE 0x20000000u   /* by its values */

/* Where a workgroup's run of the list begins: sequence, key head, row block, tile; how many tiles it has (0: none), and
 * how many the runs have that a group goes on in. */
struct KcStart {
    int b, h, rb, at, left, step, pad[2];
};
/* A group that begins in a workgroup's run and goes on in those up to w_last's (0: there is none). */
struct KcJoin {
    int w_last, q0, head, rb, rows, pad[3];
};

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
    KcStart *starts; /* of the attention's workgroups */
    KcJoin *joins;
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
    s.len = min(max(a.lens[b], 0), KC_LENGTH);
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
    int wave[4]; /* of the scanning workgroup's waves */
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
/* The last i of lo .. hi - 1 with v(i) <= x, where v(lo) is. */
template <class F>
__device__ __forceinline__ int kc_last(int lo, int hi, int x, F v) {
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v(mid) <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}
/* One workgroup finds where the attention's `grid` workgroups begin. Runs are equal shares of the list, or, where the
 * longest is then not much longer, whole groups or equal parts of groups: workgroups of one key head then walk
 * its tiles side by side, which the XCD's L2 serves. 2048 tokens over 16384, 512 groups: 555 us so, 577 with equal
 * shares (3% and 41% of L2 reads missed). */
__device__ __forceinline__ void kc_starts(const KcArgs &a, KcPlan &p, int *cnt, int grid) {
    const int pairs = a.B * a.nblk;
    auto blocks = [&](int b) { return (kc_seq(a, b).rows + KC_ROWS - 1) / KC_ROWS; };
    kc_scan(p, a.B, blocks);
    for (int i = threadIdx.x; i <= a.B; i += blockDim.x)
        cnt[i] = p.pre[i];
    __syncthreads();
    int most = 0;
    kc_scan(p, pairs, [&](int i) {
        const int c = kc_cost(a, kc_seq(a, i / a.nblk), i % a.nblk);
        most = max(most, c);
        return c;
    });
    most = (int)glint_wave_max((float)min(most, 1 << 24));
    if ((threadIdx.x & 63) == 0)
        p.wave[threadIdx.x >> 6] = most;
    __syncthreads();
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w)
        most = max(most, p.wave[w]);
    const int total = a.Hn * p.pre[pairs], groups = a.Hn * cnt[a.B];
    const int share = max(KC_SHARE, (total + grid - 1) / grid);
    const int parts = groups ? max(1, grid / groups) : 1, each_wg = (groups + grid - 1) / grid;
    const int step = (most + parts - 1) / parts;
    const bool whole = (int64_t)each_wg * step * 8 <= (int64_t)share * 9 && step >= KC_SHARE;
    auto at_group = [&](int g, KcStart &s) {
        s.b = kc_last(0, a.B, g, [&](int b) { return a.Hn * cnt[b]; });
        const int n = cnt[s.b + 1] - cnt[s.b], in = g - a.Hn * cnt[s.b];
        s.h = in / n;
        s.rb = in % n;
        const int *pre = p.pre + s.b * a.nblk;
        return a.Hn * pre[0] + s.h * (pre[a.nblk] - pre[0]) + pre[s.rb] - pre[0]; /* units before it */
    };
    for (int w = threadIdx.x; w < grid; w += blockDim.x) {
        KcStart s{0, 0, 0, 0, 0, share, {0, 0}};
        if (whole) {
            const int g = parts > 1 ? w / parts : w * each_wg;
            if (g < groups) {
                const int u = at_group(g, s);
                if (parts > 1) {
                    const int cost = p.pre[s.b * a.nblk + s.rb + 1] - p.pre[s.b * a.nblk + s.rb];
                    s.step = (cost + parts - 1) / parts;
                    s.at = w % parts * s.step;
                    s.left = max(0, min(s.step, cost - s.at));
                } else {
                    KcStart next;
                    s.left = (g + each_wg < groups ? at_group(g + each_wg, next) : total) - u;
                }
            }
        } else if ((int64_t)w * share < total) {
            const int u = w * share;
            s.left = min(share, total - u);
            s.b = kc_last(0, a.B, u, [&](int b) { return a.Hn * p.pre[b * a.nblk]; });
            const int *pre = p.pre + s.b * a.nblk;
            const int each = pre[a.nblk] - pre[0], in = u - a.Hn * pre[0];
            s.h = in / each;
            const int r = in % each + pre[0];
            s.rb = kc_last(0, a.nblk, r, [&](int i) { return pre[i]; });
            s.at = r - pre[s.rb];
        }
        a.starts[w] = s;
    }
}

union KcFrag {
    uint32_t u[4];
    glint_u32x4 v;
    kc_f16x8 f;
};
__device__ __forceinline__ uint32_t kc_uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
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

/* The exponent e of a power of two 2^(14 - e) that brings `top` (finite) under 2^15, in steps of `step`. */
__device__ __forceinline__ int ku_exponent(float top, int step) {
    const int e = max(-112, (int)(__float_as_uint(top) >> 23) - 127);
    return (e + step - 1) & -step;
}

/* The values' power of a tile, of which `top` is the largest, as KcMeta holds it; low: some token's lie below KC_SPAN of it. */
__device__ __forceinline__ uint32_t ku_values(float top, bool low, int &e) {
    const int at = ku_exponent(top, 8);
    e = max(at, -KC_BAND); /* also of a tile of zeros */
    return (uint32_t)(e + KC_EXP) | (low || (top > 0.f && (at < -KC_BAND || at > KC_BAND)) ? KC_WIDE : 0u);
}

/* The last workgroup lays out the attention's work; the others take tiles in turn. */
template <int D, bool OWN>
__global__ __launch_bounds__(KU_T, 4) void k_kv4_unpack(KcArgs A, int grid) {
    constexpr int NB = D / 64, TILE = AP_KEYS * D * 2, CH = D / 8;
    __shared__ float parents[16 * 64]; /* a copy for every lane's bank */
    __shared__ __attribute__((aligned(16))) uint16_t rows[OWN ? AP_KEYS : 1][D + 2]; /* own values, to be turned */
    __shared__ float tops[2][KU_T / 64];
    __shared__ uint32_t odds; /* KC_ODD, KC_WIDE of own values */
    __shared__ KcPlan plan;
    __shared__ int counts[KC_PAIRS + 1];
    if (blockIdx.x + 1 == gridDim.x) {
        kc_starts(A, plan, counts, grid);
        return;
    }
    for (int i = threadIdx.x; i < 16 * 64; i += KU_T)
        parents[i] = kKv4Parent[i >> 6];
    /* the list: a sequence's tiles, head after head */
    kc_scan(plan, A.B, [&](int b) {
        const KcTiles t = kc_tiles(A, kc_seq(A, b), 0, A.nblk);
        return t.np + t.nf;
    });
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int total = A.Hn * plan.pre[A.B];
    int b = 0;
    for (int u = blockIdx.x; u < total; u += gridDim.x - 1) {
        while (A.Hn * plan.pre[b + 1] <= u) /* u only grows */
            ++b;
        b = __builtin_amdgcn_readfirstlane(b);
        const int each = plan.pre[b + 1] - plan.pre[b], in = u - A.Hn * plan.pre[b];
        const int hl = in / each, i = in % each, h = A.h0 + hl;
        const KcSeq s = kc_seq(A, b);
        const KcTiles t = kc_tiles(A, s, 0, A.nblk);
        const int gap = s.len - s.nq;
        const int low = (int)max((int64_t)0, (int64_t)gap - A.bound.window + 1), high = gap + (s.rows - 1) / A.G; /* what some row sees */
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
            const float vmost = glint_wave_max(mine ? vtop : 0.f);
            bool below = false;
#pragma unroll
            for (int x = 0; x < NB; ++x)
                below |= vl[x] != 0.f && fabsf(vl[x]) < vmost * KC_SPAN;
            int ve;
            const int ke = ku_exponent(glint_wave_max(mine ? ktop : 0.f), 1);
            const uint32_t vexp = ku_values(vmost, __any(mine && below), ve);
            const float kdown = ldexpf(1.f, 14 - ke), vdown = ldexpf(1.f, 14 - ve);
            meta = KcMeta{ldexpf(1.f, ke - 14), vexp | (__any(mine && odd) ? KC_ODD : 0u)};
            if (threadIdx.x == 0)
                A.meta[slot] = meta;
            auto parent = [&](uint32_t word, int nibble) { return parents[(word >> (4 * nibble) & 15u) * 64 + lane]; };
#pragma unroll
            for (int x = 0; x < NB; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    glint_u32x4 eight;
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                        eight[z] = kc_f16pair(parent(kw[x][y], 2 * z) * (ks[x] * kdown), parent(kw[x][y], 2 * z + 1) * (ks[x] * kdown));
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
                            a[k] = parent(vw[j], 2 * k) * f;
                            z[k] = parent(vw[j], 2 * k + 1) * f;
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
        } else if constexpr (OWN) {
            /* own keys: positions s.own + 64 f ..; rows past the sequence's last are 0 */
            const int f = i - t.np < t.fsinks ? i - t.np : i - t.np + t.fskip;
            const int64_t slot = kc_slot(A, b, hl, A.max_pages + f);
            char *kt = A.tiles + slot * (2 * TILE), *vt = kt + TILE;
            const int key = s.own + f * AP_KEYS;
            const int64_t row0 = (int64_t)s.q0 + s.nq - s.len + key;
            constexpr int PER = AP_KEYS * CH / KU_T; /* 16-B chunks of a thread */
            int ke = 0, ve = 0;
            uint32_t vexp = 0;
            if (threadIdx.x == 0)
                odds = 0;
#pragma unroll 1
            for (int is_v = 0; is_v < 2; ++is_v) {
                const uint16_t *from = is_v ? A.v + row0 * A.v_st + h * A.v_sh : A.k + row0 * A.k_st + h * A.k_sh;
                const int64_t st = is_v ? A.v_st : A.k_st;
                glint_u32x4 in[PER];
                float top = 0.f, least = INFINITY; /* least: the smallest of the rows' 64-blocks' largest, but for zeros */
                bool odd = false;
#pragma unroll
                for (int x = 0; x < PER; ++x) {
                    const int r = (threadIdx.x + x * KU_T) / CH, c = (threadIdx.x + x * KU_T) % CH;
                    float block = 0.f;
                    in[x] = glint_u32x4{0, 0, 0, 0};
                    if (key + r < s.len && seen(key + r))
                        in[x] = *(const glint_u32x4 *)(from + r * st + 8 * c);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float a = fabsf(k ? glint_bf16hi(in[x][j]) : glint_bf16lo(in[x][j]));
                            if (a <= FLT_MAX) {
                                block = fmaxf(block, a);
                            } else if (is_v) { /* a key's stays: what sees it is NaN */
                                odd = true;
                                in[x][j] &= k ? 0xFFFFu : 0xFFFF0000u;
                            }
                        }
                    top = fmaxf(top, block);
                    block = kv4_max_dpp<GLINT_DPP_QUAD_1032>(block); /* of 8 lanes, a row's 64 dimensions */
                    block = kv4_max_dpp<GLINT_DPP_QUAD_2301>(block);
                    block = kv4_max_dpp<GLINT_DPP_ROW_HALF_MIRROR>(block);
                    least = block > 0.f ? fminf(least, block) : least;
                }
                top = glint_wave_max(top);
                if (lane == 0)
                    tops[is_v][wave] = top;
                __syncthreads(); /* also: the tile before has been turned */
#pragma unroll
                for (int x = 0; x < KU_T / 64; ++x)
                    top = fmaxf(top, tops[is_v][x]);
                if (odd)
                    atomicOr(&odds, KC_ODD);
                if (is_v && least < top * KC_SPAN)
                    atomicOr(&odds, KC_WIDE);
                if (is_v)
                    vexp = ku_values(top, false, ve);
                else
                    ke = ku_exponent(top, 1);
                const float down = ldexpf(1.f, 14 - (is_v ? ve : ke));
#pragma unroll
                for (int x = 0; x < PER; ++x) {
                    const int r = (threadIdx.x + x * KU_T) / CH, c = (threadIdx.x + x * KU_T) % CH;
                    glint_u32x4 eight;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        eight[j] = kc_f16pair(glint_bf16lo(in[x][j]) * down, glint_bf16hi(in[x][j]) * down);
                    if (!is_v) {
                        *(glint_u32x4 *)(kt + r * (D * 2) + 16 * ap_k_chunk<D>(r, c)) = eight;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            *(uint32_t *)&rows[r][8 * c + 2 * j] = eight[j];
                    }
                }
            }
            __syncthreads();
            if (threadIdx.x == 0)
                A.meta[slot] = KcMeta{ldexpf(1.f, ke - 14), vexp | odds};
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
typedef const __attribute__((address_space(3))) glint_u32x4 kc_lds_u32x4;

/* A wave issues in order, and a product occupies the matrix unit for 32 cycles: the vector work of one tile's
 * weights stands between the products of the next tile's scores, product by product, and operands are read
 * from LDS some products ahead. The compiler would put all products first and wait for every read, so the order
 * is fixed by scheduling barriers. */
#define KC_FIXED() __builtin_amdgcn_sched_barrier(0)

/* The scores of a tile of keys, sc; where NOW, also the weights pf (f16) and their sum l of the tile before, whose scores
 * `now` holds. */
template <int D, bool NEXT, bool NOW>
__device__ __forceinline__ void kc_scores(const ap_lds *kl, const ApRows<D> &w, ap_f32x16 (&sc)[2], ap_f32x16 (&now)[2],
                                          float factor, float base, KcFrag (&pf)[4], float &l) {
    constexpr int N = D / 8, AHEAD = 4; /* products */
    KcFrag f[AHEAD];
    auto read = [&](int n) {
        const int s = n >> 1, a = n & 1;
        f[n % AHEAD].v = *(kc_lds_u32x4 *)(kl + (w.kat[s & 3] ^ (128 * (s >> 2))) + a * 32 * D * 2);
    };
    if constexpr (NEXT) {
#pragma unroll
        for (int n = 0; n < AHEAD; ++n)
            read(n);
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                sc[a][i] = 0.f;
    }
    const kc_f16x2 ones = {(_Float16)1.f, (_Float16)1.f};
    KC_FIXED();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if constexpr (NEXT) {
            KcFrag q;
            q.v = w.q[n >> 1].v;
            sc[n & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[n % AHEAD].f, q.f, sc[n & 1], 0, 0, 0);
            KC_FIXED();
            if (n + AHEAD < N)
                read(n + AHEAD);
        }
        if constexpr (NOW) {
#pragma unroll
            for (int e = 32 / N * n; e < 32 / N * (n + 1); e += 2) { /* two elements, or four */
                const int a = e >> 4, i = e & 15;
                const float x = __builtin_amdgcn_exp2f(fmaf(now[a][i], factor, -base));
                const float y = __builtin_amdgcn_exp2f(fmaf(now[a][i + 1], factor, -base));
                const uint32_t two = kc_f16pair(x, y);
                pf[2 * a + (i >> 3)].u[(i & 7) >> 1] = two;
                l = __builtin_amdgcn_fdot2(__builtin_bit_cast(kc_f16x2, two), ones, l, false);
            }
        }
        KC_FIXED();
    }
}
/* Outputs of a tile of values, and the largest of the next tile's scores meanwhile. */
template <int D>
__device__ __forceinline__ float kc_outputs(const ap_lds *vl, ApRows<D> &w, const uint32_t (&vat)[4], const KcFrag (&pf)[4],
                                            const ap_f32x16 (&sc)[2]) {
    constexpr int N = D / 8, AHEAD = 5, PARTS = D / 32; /* products; parts of the outputs */
    KcFrag f[AHEAD];
    auto read = [&](int n) { f[n % AHEAD].v = *(kc_lds_u32x4 *)(vl + vat[n / PARTS] + n % PARTS * 32 * 128); };
#pragma unroll
    for (int n = 0; n < AHEAD; ++n)
        read(n);
    KC_FIXED();
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int s = n / PARTS, d = n % PARTS;
        w.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[n % AHEAD].f, pf[s].f, w.o[d], 0, 0, 0);
        KC_FIXED();
        if (n + AHEAD < N)
            read(n + AHEAD);
#pragma unroll
        for (int e = 32 / N * n; e < 32 / N * (n + 1); ++e)
            top = fmaxf(top, sc[e >> 4][e & 15]);
        KC_FIXED();
    }
    return top;
}

/* What a wave has to know of its 32 rows: this lane's, whether it and whether any is there; what their first and their last
 * one see up to, and this lane's. Rows before the sequence's first position see nothing, as one at -1 does; less any window
 * is an int then. */
struct KcWave {
    int row;
    bool live, any;
    int low, high, last;
};
__device__ __forceinline__ KcWave kc_wave(const KcArgs &a, const KcSeq &s, int rb, int wave, int col) {
    const int first = rb * KC_ROWS + 32 * wave, row = first + col, gap = s.len - s.nq;
    return KcWave{row, row < s.rows, first < s.rows, max(-1, gap + first / a.G), max(-1, gap + min(s.rows - 1, first + 31) / a.G),
                  row < s.rows ? max(-1, gap + row / a.G) : -1};
}
/* The place of step i's tile: pages, then own keys. */
__device__ __forceinline__ int kc_place(const KcArgs &a, const KcTiles &t, int i) {
    return i < t.np ? (i < t.psinks ? i : i + t.pskip) : a.max_pages + (i - t.np < t.fsinks ? i - t.np : i - t.np + t.fskip);
}
/* What a step has to know of its tile. */
struct KcStep {
    int key, ends; /* its first position, and the last one that it may show */
    bool want;     /* whether the wave has scores to form */
    KcMeta meta;
};
__device__ __forceinline__ KcStep kc_look(const KcArgs &a, const KcSeq &s, const KcTiles &t, const KcWave &w, int64_t slot0, int i) {
    KcStep x;
    const int to = kc_place(a, t, i);
    const bool own = i >= t.np;
    x.key = own ? s.own + (to - a.max_pages) * AP_KEYS : to * AP_KEYS;
    x.ends = own ? INT32_MAX : s.held - 1;
    x.meta = a.meta[slot0 + to];
    x.want = w.any && x.key <= min(w.high, x.ends) && (x.key + AP_KEYS - 1 > w.low - a.bound.window || x.key < a.bound.sinks);
    return x;
}
/* A row of q, its sign the scale's: the power of two that brings it to 2^14 .. 2^15 is 2^-(what is returned). */
template <int D>
__device__ __forceinline__ int kc_load_q(const KcArgs &a, const uint16_t *qr, ApFrag (&q)[D / 16], int half) {
    uint32_t high = 0;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
        q[x].v = *(const glint_u32x4 *)(qr + 16 * x + 8 * half);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[x].u[i] ^= a.q_sign;
            high = max(high, max((q[x].u[i] & 0x7FFFu) << 16, q[x].u[i] & 0x7FFF0000u));
        }
    }
    high = __float_as_uint(glint_xor32(__uint_as_float(min(high, 0x7F800000u)), GlintMax()));
    return high >= 0x7F800000u ? 0 : (int)(high >> 23) - 127 - 14;
}
/* What scores of a tile are multiplied by, `factor` being the row's part. */
__device__ __forceinline__ float kc_factor(float factor, const KcMeta &meta) { return fminf(fmaxf(factor * meta.kback, FLT_MIN), FLT_MAX); }
/* The largest kback, in bits (of two floats above 0 the larger has the larger), that leaves the wave's factors below KC_KEYS. */
__device__ __forceinline__ uint32_t kc_keys(float factor) { return kc_uniform(__float_as_uint(KC_KEYS / glint_wave_max(factor))); }
__device__ __forceinline__ bool kc_wide(const KcMeta &meta, uint32_t keys) {
    return !(meta.vexp & KC_ABSENT) && ((meta.vexp & KC_WIDE) || __float_as_uint(meta.kback) > keys);
}

/* A wide tile, from where it came: every operand as two of bf16, which has f32's range, one the other's rest: 2^-16 of each
 * element is left out. Rows `from` on of own keys and values, or the page and head of that place; the first is position `at`, and
 * past element `there` nothing is read of own ones. f is the scores' factor, keys are multiplied by kdown, q holds bf16. */
template <int D>
__device__ __forceinline__ void kc_wide_tile(const KcArgs &A, ApRows<D> &w, int h, bool own, int64_t from, int at,
                                             int last, int upto, int there, float f, float kdown, int half) {
    const int lane = threadIdx.x & 63, col = lane & 31;
    const float my_parent = kKv4Parent[lane & 15];
    auto parent = [&](uint32_t code) { return __shfl(my_parent, (int)(code & 15u), 64); };
    auto split = [](const float (&x)[8], ApFrag &hi, ApFrag &lo) { /* hi is cut off, so that it stays finite */
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t a = __float_as_uint(x[2 * j]), b = __float_as_uint(x[2 * j + 1]);
            hi.u[j] = (a >> 16) | (b & 0xFFFF0000u);
            lo.u[j] = glint_cvt_bf16x2(x[2 * j] - __uint_as_float(a & 0xFFFF0000u), x[2 * j + 1] - __uint_as_float(b & 0xFFFF0000u));
        }
    };
    ap_f32x16 sc[2];
    float x[8];
    ApFrag hi, lo;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const int r = 32 * a + col;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sc[a][i] = 0.f;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) { /* dimensions 16 n + 8 half .. of key r */
            if (own) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[e] = 0.f;
                if (r <= there)
                    kt_load8<D>(A.k + (from + r) * A.k_st + h * A.k_sh + 16 * n + 8 * half, x);
            } else {
                const uint32_t c = *(const uint32_t *)(A.k_hole + (from * KV4_PAGE + r) * (D / 2) + kv4_k_byte<D / 64>(16 * n + 8 * half));
                const float sk = A.k_absmax[(from * (D / 64) + (n >> 2)) * KV4_PAGE + r];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[e] = parent(c >> (4 * e)) * sk;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] *= kdown;
            split(x, hi, lo);
            sc[a] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi.f, w.q[n].f, sc[a], 0, 0, 0);
            sc[a] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo.f, w.q[n].f, sc[a], 0, 0, 0);
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = at + 32 * a + 8 * (i >> 2) + 4 * half + (i & 3);
            sc[a][i] = key <= upto && A.bound.sees(key, last) ? sc[a][i] * f : -INFINITY;
            top = fmaxf(top, sc[a][i]);
        }
    top = glint_xor32(top, GlintMax());
    if (top > w.m) { /* no slack: no weight is above 1 */
        const float keep = __builtin_amdgcn_exp2f(w.m - top);
        w.m = top;
        w.l *= keep;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                w.o[d][i] *= keep;
    }
    /* not a fused product: a score far from 0 then lies as far above the maximum as that says */
    const float base = w.m == -INFINITY ? 0.f : w.m;
    ApFrag ph[4], pl[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = __builtin_amdgcn_exp2f(sc[n >> 1][8 * (n & 1) + e] - base);
            w.l += x[e];
        }
        split(x, ph[n], pl[n]);
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int n = 0; n < 4; ++n) { /* keys 16 n + 4 half + 0..3, and 8 on, of dimension 32 d + col */
            const int r = 16 * n + 4 * half;
            if (own) {
                const uint16_t *v = A.v + (from + r) * A.v_st + h * A.v_sh + 32 * d + col;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int k = (e & 3) + 2 * (e & 4);
                    x[e] = r + k <= there ? __uint_as_float((uint32_t)v[k * A.v_st] << 16) : 0.f;
                }
            } else {
                const uint8_t *v = A.v_hole + (from * (D / 2) + 16 * d + (col & 15)) * KV4_PAGE + r;
                const float *sv = A.v_absmax + (from * (D / 64) + (d >> 1)) * KV4_PAGE + r;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint32_t c = *(const uint32_t *)(v + 8 * y) >> (col & 16 ? 4 : 0);
                    const glint_f32x4 scale = *(const glint_f32x4 *)(sv + 8 * y);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[4 * y + e] = parent(c >> (8 * e)) * scale[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = fabsf(x[e]) <= FLT_MAX ? x[e] : 0.f;
            split(x, hi, lo);
            w.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi.f, ph[n].f, w.o[d], 0, 0, 0);
            w.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi.f, pl[n].f, w.o[d], 0, 0, 0);
            w.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo.f, ph[n].f, w.o[d], 0, 0, 0);
        }
}

/* What the steps at .. end - 1 of a row block leave out. */
template <int D>
__device__ __forceinline__ void kc_rare(const KcArgs &A, ApRows<D> &w, const KcSeq &s, const KcTiles &tiles, const KcWave &W, int b, int h,
                                        int at, int end, bool wide, bool apart, int lane) {
    const int half = lane >> 5;
    if (wide) {
        const int64_t slot0 = kc_slot(A, b, h, 0);
        ApFrag (&q)[D / 16] = w.q;
        const int row = W.live ? W.row : 0;
        const int ex = kc_load_q<D>(A, A.q + (int64_t)(s.q0 + row / A.G) * A.q_st + ((A.h0 + h) * A.G + row % A.G) * A.q_sh, q, half);
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                q[x].u[i] = glint_cvt_bf16x2(ldexpf(glint_bf16lo(q[x].u[i]), -ex), ldexpf(glint_bf16hi(q[x].u[i]), -ex));
        const float factor = ldexpf(A.scale2, ex);
        const uint32_t keys = kc_keys(factor);
#pragma unroll 1
        for (int i = at; i < end; ++i) {
            const KcStep T = kc_look(A, s, tiles, W, slot0, i);
            if (!T.want || !kc_wide(T.meta, keys))
                continue;
            int64_t from = (int64_t)s.q0 + s.nq - s.len + T.key; /* row of the first own key, or place of the page and head */
            if (i < tiles.np)
                from = (int64_t)A.table[(int64_t)b * A.table_stride + T.key / KV4_PAGE] * A.H + A.h0 + h;
            kc_wide_tile<D>(A, w, A.h0 + h, i >= tiles.np, from, T.key, W.last, min(W.last, T.ends), min(W.high - T.key, AP_KEYS - 1),
                            kc_factor(factor, T.meta), 1.f / T.meta.kback, half);
        }
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
                    if (!A.bound.sees(key, W.last))
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
                for (int key = first; key < min(first + AP_KEYS, min(W.high + 1, s.len)); ++key) {
                    const uint16_t *from = A.v + ((int64_t)s.q0 + s.nq - s.len + key) * A.v_st + (A.h0 + h) * A.v_sh + 32 * d + 4 * half;
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const uint32_t v = from[8 * (x >> 2) + (x & 3)];
                        if ((v & 0x7F80u) == 0x7F80u && A.bound.sees(key, W.last))
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
}

/* A workgroup's run. Returns whether the wave left something out: wide tiles and values that are not finite, which a pass that
 * is RARE takes at the end of each row block (kc_rare). */
template <int D, bool RARE>
__device__ __forceinline__ bool kc_pass(const KcArgs &A, int me, char (&k0t)[AP_KEYS * D * 2], char (&k1t)[AP_KEYS * D * 2],
                                        char (&v0t)[AP_KEYS * D * 2], char (&v1t)[AP_KEYS * D * 2]) {
    constexpr int TILE = AP_KEYS * D * 2, LOADS = TILE / (16 * KC_T);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    bool rare = false;
    int left = A.starts[me].left; /* of this workgroup's run */
    if (left == 0) {
        if (threadIdx.x == 0)
            A.joins[me].w_last = 0;
        return false;
    }
    int b = A.starts[me].b, h = A.starts[me].h, rb = A.starts[me].rb, at = A.starts[me].at;

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
        const KcWave W = kc_wave(A, s, rb, wave, col);
        const int row = W.row, head = (A.h0 + h) * A.G, wave_low = W.low, wave_high = W.high;
        const bool live = W.live, wave_live = W.any;
        w.m = -INFINITY;
        w.l = 0.f;
        w.last = W.last;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                w.o[d][i] = 0.f;
        bool apart = false;
        int oexp = -4096; /* the outputs are 2^(14 - oexp) times themselves: the last tile's power */
        bool wide = false; /* there are wide tiles among those that the wave sees */
        if (at < end) {
            const int64_t slot0 = kc_slot(A, b, h, 0);
            const uint32_t my = threadIdx.x * 16;
            auto tile_of = [&](int i) {
                return __builtin_amdgcn_make_buffer_rsrc((void *)(A.tiles + (slot0 + kc_place(A, tiles, i)) * (2 * TILE)), (short)0, 2 * TILE,
                                                         GLINT_BUF_DWORD3);
            };
            auto fetch_k = [&](int i, ap_lds *kt) {
                const __amdgpu_buffer_rsrc_t r = tile_of(i);
#pragma unroll
                for (int x = 0; x < LOADS; ++x)
                    ap_dma(r, kt + (x * KC_T + wave * 64) * 16, my, x * (KC_T * 16));
            };
            auto fetch_v = [&](int i, ap_lds *vt) {
                const __amdgpu_buffer_rsrc_t r = tile_of(i);
#pragma unroll
                for (int x = 0; x < LOADS; ++x)
                    ap_dma(r, vt + (x * KC_T + wave * 64) * 16, my, TILE + x * (KC_T * 16));
            };
            KcStep T, N;
            auto look = [&](int i, KcStep &X) { X = kc_look(A, s, tiles, W, slot0, i); };
            ap_lds *const ka = (ap_lds *)(at & 1 ? k1t : k0t);
            __syncthreads(); /* the last group's tiles are read */
            fetch_k(at, ka);
            look(at, T);
            /* q as f16, scaled to 2^14 .. 2^15 by a power of two of the row's */
            const uint16_t *qr = A.q + (int64_t)(s.q0 + (live ? row / A.G : 0)) * A.q_st + (head + (live ? row % A.G : 0)) * A.q_sh;
            const int ex = kc_load_q<D>(A, qr, w.q, half);
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w.q[x].u[i] = kc_f16pair(ldexpf(glint_bf16lo(w.q[x].u[i]), -ex), ldexpf(glint_bf16hi(w.q[x].u[i]), -ex));
            const float factor = ldexpf(A.scale2, ex);

            /* Step i weighs tile i, whose scores step i - 1 has formed, and forms tile i + 1's: keys are fetched two
             * tiles ahead and values one. */
            ap_f32x16 sa[2], sb[2];
            KcFrag pf[4];
            float top = -INFINITY, l = 0.f;
            const uint32_t keys = kc_keys(factor);
            auto decide = [&](KcStep &X) { /* whether the wave takes the tile into its products */
                const bool fits = !(X.meta.vexp & (KC_ABSENT | KC_WIDE)) && __float_as_uint(X.meta.kback) <= keys;
                wide |= X.want && !fits;
                X.want = X.want && fits;
            };
            __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0);
            __syncthreads();
            decide(T);
            if (at + 1 < end)
                fetch_k(at + 1, (ap_lds *)(at & 1 ? k0t : k1t));
            fetch_v(at, (ap_lds *)(at & 1 ? v1t : v0t));
            auto largest = [&](const ap_f32x16 (&sc)[2]) {
                float m = -INFINITY;
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        m = fmaxf(m, sc[a][i]);
                return m;
            };
            auto first = [&](ap_f32x16 (&sc)[2]) {
                if (T.want) {
                    kc_scores<D, true, false>(ka, w, sc, sc, 0.f, 0.f, pf, l);
                    top = largest(sc);
                }
            };
            auto step = [&](int i, ap_f32x16 (&sc)[2], ap_f32x16 (&next)[2], ap_lds *vt, ap_lds *kn, ap_lds *vn, ap_lds *knn) {
                const bool more = i + 1 < end;
                if (more)
                    look(i + 1, N);
                __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0); /* this wave's part of what was fetched a step before */
                __syncthreads();
                if (i + 2 < end)
                    fetch_k(i + 2, knn); /* over tile i's, which every wave has left */
                if (more)
                    fetch_v(i + 1, vn);
                N.want = more && N.want;
                decide(N);
                apart |= (T.meta.vexp & (KC_ODD | KC_ABSENT)) == KC_ODD;
                if (T.want) {
                    const float f = kc_factor(factor, T.meta);
                    if (T.key + AP_KEYS - 1 > min(wave_low, T.ends) ||
                        !(T.key > wave_high - A.bound.window || T.key + AP_KEYS <= A.bound.sinks)) { /* what a row does not see */
                        const int from = T.key + 4 * half, upto = min(w.last, T.ends);
#pragma unroll
                        for (int a = 0; a < 2; ++a)
#pragma unroll
                            for (int x = 0; x < 16; ++x) { /* element x of part a is key 32 a + 8 (x / 4) + 4 half + x % 4 */
                                const int key = from + 32 * a + 8 * (x >> 2) + (x & 3);
                                sc[a][x] = key <= upto && A.bound.sees(key, w.last) ? sc[a][x] : -INFINITY;
                            }
                        top = largest(sc);
                    }
                    top = glint_xor32(top, GlintMax()) * f;
                    const bool up = top > w.m + AP_SLACK; /* a row's own test: its bits depend on no other row */
                    const int ve = (int)(T.meta.vexp & 0xFFFFu) - KC_EXP;
                    /* The outputs go to the tile's power, up or down, and not the weights, whose f16 has no bits to spare:
                     * at 2^-17 of the largest value met, weights times 2^-24 lost half of themselves. They do once the weights are
                     * formed: without this branch between them and the products the compiler copies the weights, 2048 tokens over
                     * 16384 559 us so, 592 with it before the weights. */
                    const bool other = __any(up) || ve != oexp;
                    float keep = 1.f;
                    if (other) {
                        const float mn = up ? top : w.m;
                        keep = __builtin_amdgcn_exp2f(w.m - (mn == -INFINITY ? 0.f : mn));
                        w.m = mn;
                        l *= keep;
                        keep *= ldexpf(1.f, max(oexp - ve, -300));
                        oexp = ve;
                    }
                    const float base = w.m == -INFINITY ? 0.f : w.m - KC_UP;
                    if (N.want)
                        kc_scores<D, true, true>(kn, w, next, sc, f, base, pf, l);
                    else
                        kc_scores<D, false, true>(kn, w, next, sc, f, base, pf, l);
                    if (other) {
#pragma unroll
                        for (int d = 0; d < D / 32; ++d)
#pragma unroll
                            for (int x = 0; x < 16; ++x)
                                w.o[d][x] *= keep;
                    }
                    top = kc_outputs<D>(vt, w, vat, pf, next);
                } else if (N.want) {
                    kc_scores<D, true, false>(kn, w, next, sc, 0.f, 0.f, pf, l);
                    top = largest(next);
                }
                T = N;
            };
            if (at & 1)
                first(sb);
            else
                first(sa);
            int i = at;
            if (at & 1) {
                step(i, sb, sa, (ap_lds *)v1t, (ap_lds *)k0t, (ap_lds *)v0t, (ap_lds *)k1t);
                ++i;
            }
            for (; i < end; i += 2) {
                step(i, sa, sb, (ap_lds *)v0t, (ap_lds *)k1t, (ap_lds *)v1t, (ap_lds *)k0t);
                if (i + 1 < end)
                    step(i + 1, sb, sa, (ap_lds *)v1t, (ap_lds *)k0t, (ap_lds *)v0t, (ap_lds *)k1t);
            }
            /* to the values' own size and the softmax's weights, so that no sum is far above the values */
            w.l = ldexpf(l, -(int)KC_UP);
            const float back = ldexpf(1.f, max(oexp - 14 - (int)KC_UP, -300));
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    w.o[d][x] *= back;
        }

        if (wide || apart) {
            if constexpr (RARE)
                kc_rare<D>(A, w, s, tiles, W, b, h, at, end, wide, apart, lane);
            else
                rare = true;
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
        if (left == 0) {
            if (at == 0 && take < cost) {
                const int step = A.starts[me].step, w_last = me + (cost - take + step - 1) / step;
                if (threadIdx.x == 0)
                    A.joins[me] = KcJoin{w_last, s.q0, head, rb, s.rows, {0, 0, 0}};
            } else if (threadIdx.x == 0) {
                A.joins[me].w_last = 0;
            }
            break;
        }
        at = 0;
        for (;;) { /* the next group that has rows */
            if (++rb == A.nblk) {
                rb = 0;
                if (++h == A.Hn) {
                    h = 0;
                    ++b;
                }
            }
            if (rb * KC_ROWS < kc_seq(A, b).rows)
                break;
            rb = A.nblk - 1; /* no further block of this head has */
        }
    }
    return rare;
}

template <int D>
__global__ __launch_bounds__(KC_T, 2) void k_kv4_chunk(KcArgs A) {
    constexpr int TILE = AP_KEYS * D * 2;
    /* arrays of their own, so that reads of one do not wait for loads into the other */
    __shared__ __attribute__((aligned(16))) char k0t[TILE], k1t[TILE], v0t[TILE], v1t[TILE];
    __shared__ int left_out;
    /* neighbours in the list share keys: they go to one XCD, a workgroup's being its index modulo 8 */
    const int grid = gridDim.x, me = grid & 7 ? (int)blockIdx.x : ((int)blockIdx.x & 7) * (grid >> 3) + ((int)blockIdx.x >> 3);
    if (threadIdx.x == 0)
        left_out = 0;
    __syncthreads();
    if (kc_pass<D, false>(A, me, k0t, k1t, v0t, v1t))
        left_out = 1;
    __syncthreads();
    /* A run that left something out is gone through once more. What is rare has registers of its own so: at the end of each row
     * block it cost the loop 2048 tokens over 16384 561 us where this takes 532, as a launch of its own 549. The arguments are
     * read again for the same reason. */
    if (left_out) {
        typedef const __attribute__((address_space(4))) KcArgs KernArgs;
        KernArgs *again = (KernArgs *)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(again));
        kc_pass<D, true>(*(const KcArgs *)again, me, k0t, k1t, v0t, v1t);
    }
}

/* The group that begins in workgroup w's run and ends in a later one's: its parts, added in the list's order. Blocks
 * (w, y); a block takes KJ_ROWS rows, D / 4 lanes one, each 4 dimensions. */
#define KJ_T 256
#define KJ_ROWS 8
template <int D>
__global__ __launch_bounds__(KJ_T) void k_kv4_chunk_join(KcArgs A) {
    constexpr int LANES = D / 4, AHEAD = 4;
    const int me = blockIdx.x;
    const KcJoin J = A.joins[me];
    if (J.w_last == 0 || J.rb * KC_ROWS + (int)blockIdx.y * KJ_ROWS >= J.rows)
        return;
    const int lane = threadIdx.x % LANES, parts = J.w_last - me + 1;
    for (int r = threadIdx.x / LANES; r < KJ_ROWS; r += KJ_T / LANES) {
        const int in = blockIdx.y * KJ_ROWS + r, row = J.rb * KC_ROWS + in;
        const bool live = row < J.rows;
        auto slot = [&](int p) { return (int64_t)(2 * (me + p) + (p == 0)) * KC_ROWS + in; };
        float m = -INFINITY, l = 0.f;
        glint_f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int p0 = 0; p0 < parts; p0 += AHEAD) {
            glint_f32x4 v[AHEAD];
            glint_f32x2 ml[AHEAD];
#pragma unroll
            for (int p = 0; p < AHEAD; ++p) {
                ml[p] = glint_f32x2{-INFINITY, 0.f};
                v[p] = glint_f32x4{0.f, 0.f, 0.f, 0.f};
                if (live && p0 + p < parts) {
                    ml[p] = *(const glint_f32x2 *)(A.sums + slot(p0 + p) * 2);
                    v[p] = *(const glint_f32x4 *)(A.part + slot(p0 + p) * D + 4 * lane);
                }
            }
            float top = m;
#pragma unroll
            for (int p = 0; p < AHEAD; ++p)
                top = fmaxf(top, ml[p].x);
            const float base = top == -INFINITY ? 0.f : top, keep = __builtin_amdgcn_exp2f(m - base);
            m = top;
            l *= keep;
            o *= keep;
#pragma unroll
            for (int p = 0; p < AHEAD; ++p) {
                const float f = __builtin_amdgcn_exp2f(ml[p].x - base);
                l = fmaf(f, ml[p].y, l);
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    o[x] = fmaf(f, v[p][x], o[x]);
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (live)
            *(glint_u32x2 *)(A.out + ((int64_t)(J.q0 + row / A.G) * A.Hq + J.head + row % A.G) * D + 4 * lane) =
                glint_u32x2{glint_cvt_bf16x2(o[0] * inv, o[1] * inv), glint_cvt_bf16x2(o[2] * inv, o[3] * inv)};
    }
}

/* How a call is cut into launches: sequences and key heads of one, its tiles a sequence and head, workgroups; and the
 * scratch memory's parts. No sequence fits: seqs is 0. */
struct KcCut {
    int64_t seqs;
    int heads, slots, nblk, grid;
    int unpack; /* workgroups of k_kv4_unpack */
    int64_t sums, starts, joins, meta, tiles, bytes; /* offsets; all of it */
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
    c.starts = c.sums + (int64_t)c.grid * 2 * KC_ROWS * 2 * 4;
    c.joins = c.starts + c.grid * (int64_t)sizeof(KcStart);
    c.meta = c.joins + c.grid * (int64_t)sizeof(KcJoin);
    const int64_t slots = c.seqs * c.heads * c.slots;
    c.unpack = (int)std::min<int64_t>(4 * glint_cu_count(), slots) + 1;
    c.tiles = (c.meta + slots * (int64_t)sizeof(KcMeta) + 255) & -256;
    c.bytes = c.tiles + slots * 4 * AP_KEYS * D;
    return c;
}
/* Calls that glint_kv4_attend.hip's kernel takes, whose waves decode the pages that they read and whose start is one
 * launch: few rows, or few products in all (as far as the call's bounds say). us, there against here, 8 key heads of
 * 128 dimensions:
 *   rows of a key head       128         192         256        512        1024
 *   1 sequence of 4000       20, 40      29, 49      27, 49     34, 68     60, 72
 *   1 sequence of 16000      37, 68      55, 98      61, 116    104, 101   190, 132
 *   2 sequences of 16000     60, 136     94, 112     101, 116   195, 146   376, 198
 *   8 sequences of 1000      26, 47      35, 55      45, 58     85, 57     159, 66
 *   8 sequences of 4000      61, 102     94, 95      118, 100   225, 129   436, 182
 *   8 sequences of 16000     205, 330    296, 341    389, 353   766, 467   1538, 725
 *   32 sequences of 1000     80, 89      119, 82     155, 85    302, 131   597, 216
 * and of 64 dimensions 1 of 16000 24, 49; 33, 71; 36, 79; 58, 75; 109, 94 and 8 of 4000 36, 67; 53, 67; 66, 69; 130, 88; 247, 129. */
static bool kc_few(int B, int max_q, int H, int G, int D, int max_pages) {
    const int64_t rows = (int64_t)max_q * G;
    return rows <= 192 || (double)rows * B * H * max_pages * D < 0x1p26; /* a double: the product may pass 2^63 */
}
static bool kc_shape(int B, int max_q, int Hq, int H, int D, int max_pages) {
    return B >= 0 && max_q >= 1 && H >= 1 && Hq >= H && Hq % H == 0 && Hq <= 65535 && (D == 64 || D == 128) &&
           max_pages >= 1 && max_pages <= 1 << 24 && (int64_t)max_q * (Hq / H) <= (int64_t)KC_PAIRS * KC_ROWS;
}

GLINT_API int64_t glint_kv4_attend_chunk_scratch(int B, int max_q, int Hq, int H, int D, int max_pages, int own) {
    if (!kc_shape(B, max_q, Hq, H, D, max_pages))
        return -2;
    if (B == 0 || (!own && kc_few(B, max_q, H, Hq / H, D, max_pages)))
        return 0;
    const KcCut c = kc_cut(B, max_q, H, Hq / H, D, max_pages, own != 0);
    return c.seqs ? c.bytes : -2;
}

template <int D>
static void kc_run(const KcArgs &a, const KcCut &c, hipStream_t stream) {
    if (a.k)
        k_kv4_unpack<D, true><<<c.unpack, KU_T, 0, stream>>>(a, c.grid);
    else
        k_kv4_unpack<D, false><<<c.unpack, KU_T, 0, stream>>>(a, c.grid);
    k_kv4_chunk<D><<<c.grid, KC_T, 0, stream>>>(a);
    k_kv4_chunk_join<D><<<dim3(c.grid, KC_ROWS / KJ_ROWS), KJ_T, 0, stream>>>(a);
}

GLINT_API int glint_kv4_attend_chunk(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq,
                                     const uint8_t *k_hole, const float *k_absmax, const uint8_t *v_hole,
                                     const float *v_absmax, int64_t pages, const int32_t *table, int64_t table_stride,
                                     int max_pages, const int32_t *lens, const int32_t *cu_q, int B, int max_q, int Hq, int H,
                                     int D, const uint16_t *k, int64_t k_stride_t, int64_t k_stride_h, const uint16_t *v,
                                     int64_t v_stride_t, int64_t v_stride_h, float scale, int window, int sinks,
                                     uint16_t *out, void *scratch, int64_t scratch_bytes, struct ihipStream_t *stream) {
    if (!q || !k_hole || !k_absmax || !v_hole || !v_absmax || !table || !lens || !out || !k != !v)
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
    if (!k && kc_few(B, max_q, H, Hq / H, D, max_pages))
        return glint_kv4_attend_window(q, q_stride_t, q_stride_h, Tq, k_hole, k_absmax, v_hole, v_absmax, pages, table,
                                       table_stride, max_pages, lens, cu_q, B, max_q, Hq, H, D, scale, window, sinks, out, stream);
    if (!scratch)
        return -1;
    const float scale2 = fabsf(scale) * 1.44269504088896341f;
    const KcCut c = kc_cut(B, max_q, H, Hq / H, D, max_pages, k != nullptr);
    if (!c.seqs || scratch_bytes < c.bytes)
        return -2;
    char *const mem = (char *)scratch;
    KcArgs a{q, q_stride_t, q_stride_h, Tq, k_hole, v_hole, k_absmax, v_absmax, pages, table, table_stride, max_pages, lens,
             cu_q, k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, B, max_q, Hq, H, Hq / H, c.nblk, 0, 0, c.slots,
             scale2 < FLT_MIN ? FLT_MIN : scale2, scale < 0.f ? 0x80008000u : 0u, out,
             {window ? window : INT32_MAX, window ? sinks : 0}, (float *)mem, (float *)(mem + c.sums),
             (KcStart *)(mem + c.starts), (KcJoin *)(mem + c.joins), (KcMeta *)(mem + c.meta), mem + c.tiles};
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
                kc_run<64>(a, c, stream);
            else
                kc_run<128>(a, c, stream);
            if (hipGetLastError() != hipSuccess)
                return -3;
        }
    }
    return 0;
}
