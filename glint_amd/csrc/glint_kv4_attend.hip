/* Attention over the 4-bit cache (include/glint_serve.h).
 *
 * k_kv4_attend — the work is a list of rounds: a group is one sequence, key head and block of
 *   up to 16 query rows (the heads that share the key head, times the new tokens), and a
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
 *
 *   What bounds it: reading the cache once, 4.5 bits an element. 32 sequences of 8192 tokens, 8 heads
 *   of 128, 4 rows a head: 303 MB in 62 to 69 us, 4.4 to 4.9 TB/s, where a copy reaches 5.1. Decoding
 *   codes in LDS, its two products and 2^x take some 620 vector instructions a page and hide behind
 *   that up to 16 rows a page, which is why a group has 16 (32 rows in registers spilled: 4 sequences of
 *   8000 with 40 rows a head 57 us at best, 38 now). A product's table entries are read while the one
 *   before is multiplied (equal lengths 65 without, 62 with; ragged ones 42.5, 39). 8 waves share a
 *   table: 4 waves a workgroup were slower everywhere, by the table's filling. Short calls are bound
 *   by their start, some 5 us from the launch to the first page's loads: lengths, runs, table and
 *   page numbers one after another; one sequence of 1000 tokens takes 12.8 us.
 *   Of a bounded call too: 32 sequences of 8192 under a window of 1024 and 4 first tokens read 38 MB in 17.8 us,
 *   two to three pages a wave. */
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "kv4.h"
#include "serve_ws.h"
/* two partials of 16 rows of 128 dimensions, a maximum and a sum per CU; token scores take fewer */
#define GLINT_SPLIT_CU_FLOATS (2 * 16 * (128 + 4))
#include "tile_mfma.h"

typedef _Float16 kv4_f16x8 __attribute__((ext_vector_type(8)));
/* the value scales' place in LDS holds f16 or f32 */
typedef _Float16 kv4_lds_f16 __attribute__((may_alias));
typedef kv4_f16x8 kv4_lds_f16x8 __attribute__((may_alias));
typedef float kv4_lds_f32 __attribute__((may_alias));
typedef glint_f32x4 kv4_lds_f32x4 __attribute__((may_alias));

#define KA_WAVES 8
#define KA_T (64 * KA_WAVES)
#define KA_ROWS 16 /* of q in a group */
/* What turning to a group costs, in pages: its queries, its meeting in LDS, a join. Time at 0, 8, 16: 48
 * sequences of 1 to 4097 tokens and 10 heads 50, 39, 39 us; 64 of 1 to 2000, 8 heads of one query head
 * each, 35, 30, 32; 16 of 1 to 3001 with 4 new tokens 18, 14, 15; 4 of 8000 with 40 rows a head 38, 38,
 * 34; 32 equal lengths 65 whatever it is. */
#define KA_SWITCH 8
#define KA_COPIES 32 /* of an entry; entries are 64 words apart, so that an address is one byte permute */
#define KA_TABLE_WORDS (256 * 64)
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
    float scale2;    /* |scale| log2 e / KV4_ALPHA, above 0 */
    uint32_t q_sign; /* 0x80008000 where the scale is negative */
    uint16_t *out;
    float *part; /* two partials per workgroup; NULL: groups are not split */
    unsigned *ctr;
    int window, sinks; /* of the bounded form: positions up to a row's own that it sees, and first ones */
};

/* A sequence's rows and length, with every device value bounded. */
struct Kv4Raw {
    int q0, nq, len;
};
__device__ __forceinline__ Kv4Raw kv4_raw(const Kv4AttendArgs &a, int b) {
    Kv4Raw s{0, 0, 0};
    if (b < a.B) {
        const int64_t q0 = a.cu_q ? a.cu_q[b] : (int64_t)b * a.max_q, q1 = a.cu_q ? a.cu_q[b + 1] : q0 + a.max_q;
        const int len = a.lens[b];
        if (q0 >= 0 && q1 > q0 && q1 <= a.Tq) {
            s.q0 = (int)q0;
            s.nq = (int)(q1 - q0);
        }
        s.len = (int)min((int64_t)max(len, 0), (int64_t)a.max_pages * KV4_PAGE);
    }
    return s;
}
struct Kv4Seq : Kv4Raw {
    int rows, npages;
    int sink_pages, skip; /* of the bounded form: page i of the npages is the sequence's page i, or, past the sinks', i + skip */
    int rounds; /* of a group */
    int blocks; /* row blocks */
    int all;    /* rounds of all its groups */
    int cost;   /* of a group: KA_WAVES a round, and KA_SWITCH for turning to it */
};
template <bool BOUNDED>
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttendArgs &a, const Kv4Raw &r) {
    Kv4Seq s;
    s.q0 = r.q0;
    s.nq = r.nq;
    s.len = r.len;
    s.rows = a.G * min(s.nq, a.max_q);
    s.npages = (s.len + KV4_PAGE - 1) / KV4_PAGE;
    s.sink_pages = s.skip = 0;
    if (BOUNDED) { /* up to the page that the first row's window begins in: a page at most of what is past */
        s.sink_pages = (min(a.sinks, s.len) + KV4_PAGE - 1) / KV4_PAGE;
        s.skip = max(0, (int)(max((int64_t)0, (int64_t)s.len - s.nq - a.window + 1) / KV4_PAGE) - s.sink_pages);
        s.npages -= s.skip;
    }
    s.rounds = (s.npages + KA_WAVES - 1) / KA_WAVES;
    s.blocks = (s.rows + KA_ROWS - 1) / KA_ROWS;
    s.all = s.rounds * s.blocks * a.H;
    s.cost = s.rounds > 0 ? s.rounds * KA_WAVES + KA_SWITCH : 0;
    return s;
}
__device__ __forceinline__ int kv4_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

/* Over the four lane groups that hold one row. */
template <class F>
__device__ __forceinline__ float kv4_over_row(float v, F op) { return glint_xor32(glint_xor16(v, op), op); }

/* A power of two for value scales up to `top` (finite): 2^KA_VSTART in place of the largest. The
 * outputs so far are carried over by the factor returned. An infinite scale stays infinite under
 * any power and must not push the others out of range: it is left out of `top`. */
__device__ __forceinline__ float kv4_new_power(float top, float &down, float &limit) {
    const int e = max(-126, (int)(__float_as_uint(top) >> 23) - 127 - KA_VSTART);
    const float to = ldexpf(1.f, -e), by = to / down; /* by >= 2^-252: 0 where it underflows */
    down = to;
    limit = ldexpf(1.f, e + KA_VMAX);
    return by;
}

/* A group, or the part of it that this workgroup's run holds. */
struct Kv4Group {
    Kv4Seq s;
    int b, at;    /* the sequence, and where in its rounds the part begins */
    int ahead;    /* cost of the sequences before it */
    int h, rb;    /* key head, row block */
    int k;        /* rounds of the run ahead of it */
    int begin, n; /* first round of the group, rounds */
};
/* A part that other workgroups share: what the one that joins them has to know. */
struct Kv4Join {
    int on, w_first, w_last, rows, rb, h, q0;
};

/* A row's outputs (4 dimensions), maximum and sum, added up from parts. */
struct Kv4Sum {
    glint_f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    __device__ void add(const glint_f32x4 v, float vm, float vl) {
        const float to = fmaxf(m, vm), base = to == -INFINITY ? 0.f : to;
        const float keep = __builtin_amdgcn_exp2f(m - base), f = __builtin_amdgcn_exp2f(vm - base);
        m = to;
        l = fmaf(l, keep, f * vl);
#pragma unroll
        for (int x = 0; x < 4; ++x)
            o[x] = fmaf(o[x], keep, f * v[x]);
    }
    __device__ void add_below(const glint_f32x4 v, float vm, float vl) { /* vm <= m */
        const float f = __builtin_amdgcn_exp2f(vm - (m == -INFINITY ? 0.f : m));
        l = fmaf(f, vl, l);
#pragma unroll
        for (int x = 0; x < 4; ++x)
            o[x] = fmaf(f, v[x], o[x]);
    }
    __device__ void store(uint16_t *dst) const { /* a row that saw nothing is zero */
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *(glint_u32x2 *)dst = glint_u32x2{glint_cvt_bf16x2(o[0] * inv, o[1] * inv), glint_cvt_bf16x2(o[2] * inv, o[3] * inv)};
    }
};
template <int D>
__device__ __forceinline__ uint16_t *kv4_out(const Kv4AttendArgs &a, int q0, int h, int r) {
    return a.out + ((int64_t)(q0 + r / a.G) * a.Hq + h * a.G + r % a.G) * D;
}

/* BOUNDED: a row sees the last `window` positions up to its own and the first `sinks`. The list holds the
 * pages that a sequence's rows see, so that what lies between costs nothing, and its numbers in the table are
 * not read. */
template <int D, bool BOUNDED>
__global__ __launch_bounds__(KA_T) void k_kv4_attend(Kv4AttendArgs A) {
    constexpr int NB = D / 64;
    constexpr int ROW = D + 4; /* a row's output, then its maximum and sum */
    __shared__ __attribute__((aligned(16))) uint32_t lds[KA_TABLE_WORDS];
    __shared__ __attribute__((aligned(16))) float meet[KA_WAVES * 16 * ROW];
    __shared__ __attribute__((aligned(16))) float scales[KA_WAVES * 2 * NB * KV4_PAGE];
    __shared__ unsigned s_last[2];

    const int lane = threadIdx.x & 63, wave = kv4_uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;

    /* 64 sequences, one a lane, from `chunk` on: what follows finds its way in registers */
    int chunk = 0;
    Kv4Raw raw = kv4_raw(A, lane);
    /* The table, while they are on their way: thread t writes four copies of the entries t / 8 + 64 i. */
    static_assert(KA_T == 512 && KA_COPIES == 32, "the table's shares");
    {
        const float lo = kKv4Parent[(threadIdx.x >> 3) & 15] * KV4_ALPHA;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            union {
                _Float16 f[2];
                uint32_t u;
            } e;
            e.f[0] = (_Float16)lo;
            e.f[1] = (_Float16)(kKv4Parent[(wave >> 1) + 4 * i] * KV4_ALPHA);
            ((glint_u32x4 *)lds)[((threadIdx.x >> 3) + 64 * i) * 16 + (threadIdx.x & 7)] = glint_u32x4{e.u, e.u, e.u, e.u};
        }
    }
    auto to_chunk = [&](int b) {
        chunk = b;
        raw = kv4_raw(A, b + lane);
    };
    auto sequence = [&](int b) { /* uniform; in the chunk */
        Kv4Raw r;
        r.q0 = __builtin_amdgcn_readlane(raw.q0, b - chunk);
        r.nq = __builtin_amdgcn_readlane(raw.nq, b - chunk);
        r.len = __builtin_amdgcn_readlane(raw.len, b - chunk);
        return kv4_seq<BOUNDED>(A, r);
    };
    auto scan = [](int v) { /* of the lanes up to this one: row_shr 1, 2, 4, 8, row_bcast 15, 31 */
        v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
        return v;
    };
    /* Rows of sequences without a token are zero: sequence b is workgroup b mod grid's to fill. */
    const int per = (A.B + 63) / 64; /* sequences of a lane */
    for (int c = 0; c < per; ++c) {
        const Kv4Raw r = c ? kv4_raw(A, 64 * c + lane) : raw;
        uint64_t empty = __ballot(r.len == 0 && r.nq > 0 && (64 * c + lane) % (int)gridDim.x == (int)blockIdx.x);
        for (; empty; empty &= empty - 1) {
            const int j = __builtin_ctzll(empty);
            const int q0 = __builtin_amdgcn_readlane(r.q0, j), nq = min(__builtin_amdgcn_readlane(r.nq, j), A.max_q);
            glint_u32x2 *dst = (glint_u32x2 *)(A.out + (int64_t)q0 * A.Hq * D);
            for (int64_t i = threadIdx.x; i < (int64_t)nq * A.Hq * (D / 4); i += KA_T)
                dst[i] = glint_u32x2{0, 0};
        }
    }
    /* The list in units of cost: a group is KA_SWITCH units and KA_WAVES per round; its round j belongs to
     * the workgroup whose run holds its unit KA_SWITCH + KA_WAVES j. A workgroup takes `share` units
     * (KA_WAVES at least, so that each run inside a group holds a round of it), or, where groups are
     * not split, one group. */
    auto weight = [&](const Kv4Seq &s) { return (A.part ? s.cost : s.cost > 0 ? 1 : 0) * s.blocks * A.H; };
    int mine = 0, mine_rounds = 0;
    for (int i = 0; i < per; ++i) {
        const Kv4Seq s = kv4_seq<BOUNDED>(A, per == 1 ? raw : kv4_raw(A, lane * per + i));
        mine += weight(s);
        mine_rounds += s.all;
    }
    const int upto = scan(mine), total = __builtin_amdgcn_readlane(upto, 63);
    const int share = A.part ? max(KA_WAVES, (total + (int)gridDim.x - 1) / (int)gridDim.x) : 1;
    if ((int64_t)blockIdx.x * share >= total)
        return;
    const int upto_rounds = scan(mine_rounds);
    const int u0 = blockIdx.x * share, u1 = min(total - u0, share) + u0;
    /* the sequence that unit u lies in, the rounds before u in it, and in the sequences before it */
    auto locate = [&](int u, int &b, int &at, int &ahead, int &rounds_ahead) {
        const int owner = __builtin_ctzll(__ballot(upto > u));
        ahead = __builtin_amdgcn_readlane(upto - mine, owner);
        rounds_ahead = __builtin_amdgcn_readlane(upto_rounds - mine_rounds, owner);
        b = owner * per;
        while (true) {
            if (b < chunk || b - chunk >= 64)
                to_chunk(b);
            const Kv4Seq s = sequence(b);
            const int w = weight(s);
            if (u - ahead < w) {
                const int e = A.part ? (u - ahead) % s.cost - KA_SWITCH : 0;
                at = (A.part ? (u - ahead) / s.cost : u - ahead) * s.rounds + (max(e, 0) + KA_WAVES - 1) / KA_WAVES;
                return;
            }
            ahead += w;
            rounds_ahead += s.all;
            ++b;
        }
    };
    Kv4Group G;
    int run; /* rounds */
    {
        int before, after, b1, at1, ahead1;
        if (u1 < total)
            locate(u1, b1, at1, ahead1, after);
        else {
            after = __builtin_amdgcn_readlane(upto_rounds, 63);
            at1 = 0;
        }
        locate(u0, G.b, G.at, G.ahead, before);
        run = after + at1 - before - G.at;
        G.k = 0;
    }
    if (run == 0)
        return;
    /* completes a group whose b, at, ahead and k are set */
    auto place = [&](Kv4Group &X) {
        if (X.b < chunk || X.b - chunk >= 64)
            to_chunk(X.b);
        X.s = sequence(X.b);
        while (X.at >= X.s.all) { /* on to the sequence that it lies in */
            X.at -= X.s.all;
            X.ahead += X.s.cost * X.s.blocks * A.H;
            if (++X.b - chunk == 64)
                to_chunk(X.b);
            X.s = sequence(X.b);
        }
        const int group = X.at / X.s.rounds;
        X.begin = X.at % X.s.rounds;
        X.h = kv4_uniform(group / X.s.blocks);
        X.rb = kv4_uniform(group % X.s.blocks);
        X.n = min(X.s.rounds - X.begin, run - X.k);
    };
    place(G);
    /* The lane's rows of q. */
    glint_u32x4 qw[NB][2];
    auto load_q = [&](const Kv4Group &X) {
        const int r = X.rb * KA_ROWS + col;
        const bool live = r < X.s.rows;
        const uint16_t *qr = A.q + (int64_t)(X.s.q0 + (live ? r / A.G : 0)) * A.q_st + (X.h * A.G + (live ? r % A.G : 0)) * A.q_sh;
#pragma unroll
        for (int bb = 0; bb < NB; ++bb)
#pragma unroll
            for (int st = 0; st < 2; ++st)
                qw[bb][st] = *(const glint_u32x4 *)(qr + bb * 64 + 16 * g + 8 * st);
    };
    load_q(G); /* on its way while the pages are found */
    /* This wave's pages of the run's next rounds, from group X's first on, one a lane: as many as the
     * chunk's sequences hold, 64 at most. A page that is not there, past the sequence's end or not in
     * the pool, is read as the pool's first page and seen by nobody: its lane holds -1. */
    int pids, window, window_n; /* the window's first round in the run, its length */
    auto open_window = [&](int b, int at, int k) {
        if (b < chunk || b - chunk >= 48)
            to_chunk(b);
        const int all = lane >= b - chunk ? kv4_seq<BOUNDED>(A, raw).all : 0;
        const int sum = scan(all) - at; /* rounds from here to the lane's sequence's end */
        int j = b - chunk;                /* the lane whose sequence holds this lane's round */
        if (run - k > __builtin_amdgcn_readlane(sum, j)) {
            j = 0;
#pragma unroll
            for (int step = 32; step; step >>= 1)
                j += __shfl(sum, j + step - 1, 64) <= lane ? step : 0;
        }
        /* every lane reads the others before any condition on its own */
        const int sum_j = __shfl(sum, j, 64);
        const Kv4Raw r{0, __shfl(raw.nq, j, 64), __shfl(raw.len, j, 64)};
        const bool in = lane < run - k && lane < sum_j;
        const Kv4Seq s = kv4_seq<BOUNDED>(A, r);
        const int in_seq = lane - (sum_j - s.all);
        const int pg = in_seq % max(s.rounds, 1) * KA_WAVES + wave;
        const int at_page = BOUNDED && pg >= s.sink_pages ? pg + s.skip : pg;
        pids = in && pg < s.npages ? A.table[(int64_t)(chunk + j) * A.table_stride + at_page] : -1;
        pids = pids < A.pages ? pids : -1;
        window = k;
        window_n = __builtin_popcountll(__ballot(in));
    };
    open_window(G.b, G.at, 0);

    const uint32_t lane4 = (uint32_t)(lane & (KA_COPIES - 1)) * 4;
    auto pair = [&](uint32_t word, int byte) { /* byte << 8 | lane4 */
        return *(const uint32_t *)((const char *)lds + __builtin_amdgcn_perm(word, lane4, 0x0C0C0000u | ((4u + byte) << 8)));
    };
    float *sl = scales + wave * (2 * NB * KV4_PAGE);

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
    auto page = [&](int k, int h) { /* of the run's round k; whether it is there */
        const int pid = __builtin_amdgcn_readlane(pids, k - window);
        ph = (int64_t)max(pid, 0) * A.H + h;
        return pid >= 0;
    };
    __syncthreads(); /* the table is written */
    bool there = page(0, G.h);
    load_k();
    load_v();

    Kv4Join join0{0}, join1{0}; /* of this workgroup's slot 0 and slot 1 */
    for (;;) {
        const Kv4Seq &s = G.s;
        Kv4Group N = G; /* the group after this one */
        N.k = G.k + G.n;
        N.at = G.at + G.n;
        const bool more_groups = N.k < run;
        if (more_groups)
            place(N);

        /* this lane's row of q as f16 operands, scaled to 2^14 .. 2^15 by a power of two that goes
         * into the row's score factor */
        Kv4Frag qf[NB][2];
        const int my_row = G.rb * KA_ROWS + col;
        const int last = my_row < s.rows ? s.len - s.nq + my_row / A.G : -1; /* the last position that it sees */
        uint32_t high = 0;
#pragma unroll
        for (int bb = 0; bb < NB; ++bb)
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    high = max(high, max((qw[bb][st][x] & 0x7FFFu) << 16, qw[bb][st][x] & 0x7FFF0000u));
        high = __float_as_uint(kv4_over_row(__uint_as_float(min(high, 0x7F800000u)), GlintMax())); /* inf for NaN */
        const int ex = high >= 0x7F800000u ? 0 : (int)(high >> 23) - 127 - 14;
#pragma unroll
        for (int bb = 0; bb < NB; ++bb)
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t w = qw[bb][st][x] ^ A.q_sign;
                    qf[bb][st].f[2 * x] = (_Float16)ldexpf(glint_bf16lo(w), -ex);
                    qf[bb][st].f[2 * x + 1] = (_Float16)ldexpf(glint_bf16hi(w), -ex);
                }
        const float factor = fmaxf(ldexpf(A.scale2, ex), FLT_MIN); /* above 0: -inf stays -inf */

        glint_f32x4 o[D / 16];
        float m = -INFINITY, l = 0.f, vdown[NB], vlimit[NB];
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            o[d] = glint_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int bb = 0; bb < NB; ++bb) {
            vdown[bb] = 0x1p126f;
            vlimit[bb] = 0x1p-111f;
        }
        auto carry = [&](int bb, float by) { /* block bb's outputs, to another power */
#pragma unroll
            for (int d = 4 * bb; d < 4 * bb + 4; ++d)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    o[d][x] *= by;
        };

        for (int i = 0; i < G.n; ++i) {
            /* a page that nobody sees lies past every row's last position */
            int pg = there ? (G.begin + i) * KA_WAVES + wave : KA_FAR;
            if (BOUNDED && there && pg >= s.sink_pages)
                pg += s.skip;
            /* The run's last page is loaded again: without a branch around them the next page's
             * loads can be counted, and this page's waits leave them in flight. */
            const int k = G.k + i + 1;
            if (k < run) {
                if (k - window == window_n) {
                    open_window(i + 1 < G.n ? G.b : N.b, i + 1 < G.n ? G.at + i + 1 : N.at, k);
                    __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0); /* here, not where the branch joins */
                }
                there = page(k, i + 1 < G.n ? G.h : N.h);
            }
            /* A whole page lies below every row's last position: nothing of it is masked, and the
             * rows have one power for its value scales, which go to LDS scaled and rounded to f16.
             * Of another page they go there as they are. Behind a page that rows saw in part, as a bound's first
             * ones, their powers may differ: then every page is another one. */
            bool whole = (pg + 1) * KV4_PAGE <= s.len - s.nq + 1;
            if (BOUNDED) {
                whole = whole && (pg * KV4_PAGE >= s.len - A.window || (pg + 1) * KV4_PAGE <= A.sinks);
#pragma unroll
                for (int bb = 0; bb < NB; ++bb)
                    whole = whole && !__any(__float_as_int(vdown[bb]) != __builtin_amdgcn_readfirstlane(__float_as_int(vdown[bb])));
            }
            glint_f32x4 sc[4]; /* scores, without the row's factor */
            if (pg != KA_FAR) {
#pragma unroll
                for (int bb = 0; bb < NB; ++bb) {
                    sl[bb * KV4_PAGE + lane] = sw[bb];
                    const float v = sw[NB + bb];
                    if (whole) {
                        if (__any(v >= vlimit[bb])) {
                            const float top = glint_wave_max(v < INFINITY ? v : 0.f);
                            if (top >= vlimit[bb])
                                carry(bb, kv4_new_power(top, vdown[bb], vlimit[bb]));
                        }
                        ((kv4_lds_f16 *)(sl + (NB + bb) * KV4_PAGE))[lane] = (_Float16)(v * vdown[bb]);
                    } else {
                        ((kv4_lds_f32 *)sl)[(NB + bb) * KV4_PAGE + lane] = v;
                    }
                }

                constexpr int STEPS = 2 * NB; /* products of a score */
                uint32_t e[2][4];
                auto entries = [&](int n) {
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        e[n & 1][x] = pair(kw[n / STEPS][n % STEPS], x);
                };
                entries(0);
                glint_f32x4 c[NB];
#pragma unroll
                for (int n = 0; n < 4 * STEPS; ++n) {
                    const int a = n / STEPS, bb = n % STEPS >> 1, st = n & 1;
                    if (n + 1 < 4 * STEPS)
                        entries(n + 1);
                    Kv4Frag f;
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        f.u[x] = e[n & 1][x];
                    if (st == 0)
                        c[bb] = glint_f32x4{0.f, 0.f, 0.f, 0.f};
                    c[bb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.f, qf[bb][st].f, c[bb], 0, 0, 0);
                    if (st == 1) {
                        const glint_f32x4 kscale = *(const glint_f32x4 *)(sl + bb * KV4_PAGE + 16 * g + 4 * a);
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            sc[a][x] = bb ? fmaf(c[bb][x], kscale[x], sc[a][x]) : c[bb][x] * kscale[x];
                    }
                }
            }
            load_k();
            if (pg != KA_FAR) {
                const int t0 = pg * KV4_PAGE + 16 * g;
                auto seen = [&](int t) { return t <= last && (!BOUNDED || t > last - A.window || t < A.sinks); };
                if (!whole) { /* what the row does not see */
#pragma unroll
                    for (int a = 0; a < 4; ++a)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            sc[a][x] = seen(t0 + 4 * a + x) ? sc[a][x] : -INFINITY;
                }

                /* softmax weights */
                float top = -INFINITY;
#pragma unroll
                for (int a = 0; a < 4; ++a)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        top = fmaxf(top, sc[a][x]);
                top = kv4_over_row(top, GlintMax()) * factor;
                if (__any(top > m)) {
                    const float mn = fmaxf(m, top);
                    const float keep = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
                    m = mn;
                    l *= keep;
#pragma unroll
                    for (int bb = 0; bb < NB; ++bb)
                        carry(bb, keep);
                }
                const float base = m == -INFINITY ? 0.f : m;
                float sum = 0.f;
#pragma unroll
                for (int a = 0; a < 4; ++a)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        sc[a][x] = __builtin_amdgcn_exp2f(fmaf(sc[a][x], factor, -base));
                        sum += sc[a][x];
                    }
                l += sum;

                /* times the value scales, as f16 */
                Kv4Frag pf[NB][2];
                if (whole) {
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        kv4_f16x8 w;
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            w[x] = (_Float16)sc[2 * st + (x >> 2)][x & 3];
#pragma unroll
                        for (int bb = 0; bb < NB; ++bb)
                            pf[bb][st].f =
                                w * *(const kv4_lds_f16x8 *)((const kv4_lds_f16 *)(sl + (NB + bb) * KV4_PAGE) + 16 * g + 8 * st);
                    }
                } else {
#pragma unroll
                    for (int bb = 0; bb < NB; ++bb) {
                        glint_f32x4 vscale[4];
                        float any = 0.f, finite = 0.f;
#pragma unroll
                        for (int a = 0; a < 4; ++a) {
                            vscale[a] = *(const kv4_lds_f32x4 *)(sl + (NB + bb) * KV4_PAGE + 16 * g + 4 * a);
#pragma unroll
                            for (int x = 0; x < 4; ++x) { /* an unseen place counts as 0, whatever it holds */
                                const float v = seen(t0 + 4 * a + x) ? vscale[a][x] : 0.f;
                                vscale[a][x] = v;
                                any = fmaxf(any, v);
                                finite = fmaxf(finite, v < INFINITY ? v : 0.f);
                            }
                        }
                        if (__any(any >= vlimit[bb])) { /* outside f16's range under some row's power */
                            finite = kv4_over_row(finite, GlintMax());
                            if (BOUNDED) { /* columns without a row go with the largest */
                                const float most = glint_wave_max(finite);
                                finite = last < 0 ? most : finite;
                            }
                            if (finite >= vlimit[bb])
                                carry(bb, kv4_new_power(finite, vdown[bb], vlimit[bb]));
                        }
#pragma unroll
                        for (int a = 0; a < 4; ++a)
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                pf[bb][a >> 1].f[4 * (a & 1) + x] = (_Float16)(sc[a][x] * (vscale[a][x] * vdown[bb]));
                    }
                }

                    /* outputs: a product's table entries are read while the one before is multiplied */
                uint32_t e[2][8];
                auto entries = [&](int n) {
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        e[n & 1][x] = pair(vw[n >> 1][2 * (n & 1) + (x >> 2)], x & 3);
                };
                entries(0);
#pragma unroll
                for (int n = 0; n < D / 16; ++n) {
                    const int p = n >> 1, st = n & 1;
                    if (n + 1 < D / 16)
                        entries(n + 1);
                    Kv4Frag lo, hi;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        lo.u[x] = __builtin_amdgcn_perm(e[n & 1][2 * x + 1], e[n & 1][2 * x], 0x05040100u);
                        hi.u[x] = __builtin_amdgcn_perm(e[n & 1][2 * x + 1], e[n & 1][2 * x], 0x07060302u);
                    }
                    o[2 * p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo.f, pf[p >> 1][st].f, o[2 * p], 0, 0, 0);
                    o[2 * p + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi.f, pf[p >> 1][st].f, o[2 * p + 1], 0, 0, 0);
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
        const float sum = kv4_over_row(l, GlintAdd());
        __syncthreads(); /* the previous group's rows are read */
        float *row = meet + (wave * KA_ROWS + col) * ROW;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            const float back = 1.f / vdown[d >> 2] * (1.f / KV4_ALPHA); /* a power of two, inverted exactly */
            *(glint_f32x4 *)(row + 16 * d + 4 * g) = glint_f32x4{o[d][0] * back, o[d][1] * back, o[d][2] * back, o[d][3] * back};
        }
        if (g == 0) {
            row[D] = m;
            row[D + 1] = sum;
        }
        __syncthreads();
        for (int t = threadIdx.x; t < KA_ROWS * (D / 4); t += KA_T) {
            const int c = t / (D / 4), d = 4 * (t % (D / 4));
            const int r = G.rb * KA_ROWS + c;
            if (r >= s.rows)
                continue;
            Kv4Sum z;
#pragma unroll
            for (int w = 0; w < KA_WAVES; ++w)
                z.m = fmaxf(z.m, meet[(w * KA_ROWS + c) * ROW + D]);
#pragma unroll
            for (int w = 0; w < KA_WAVES; ++w) {
                const float *wr = meet + (w * KA_ROWS + c) * ROW;
                z.add_below(*(const glint_f32x4 *)(wr + d), wr[D], wr[D + 1]);
            }
            if (whole_group) {
                z.store(kv4_out<D>(A, s.q0, G.h, r) + d);
            } else {
                float *dst = A.part + ((int64_t)(2 * blockIdx.x + slot) * KA_ROWS + c) * ROW;
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    __hip_atomic_store(dst + d + x, z.o[x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (d == 0) {
                    __hip_atomic_store(dst + D, z.m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    __hip_atomic_store(dst + D + 1, z.l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
        }
        if (!whole_group) {
            const int first = G.ahead + (G.h * s.blocks + G.rb) * s.cost + KA_SWITCH; /* the unit of its round 0 */
            const Kv4Join J{1, first / share, (first + KA_WAVES * (s.rounds - 1)) / share, s.rows, G.rb, G.h, s.q0};
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
        /* teams of threads, one thread per 4 dimensions of a row, take the parts in turn, four loads
         * of each in flight, and meet in LDS; up to four parts are one team's */
        const int rows = min(KA_ROWS, J.rows - J.rb * KA_ROWS), items = rows * (D / 4);
        const int teams = min(KA_T / items, (J.w_last - J.w_first + 4) >> 2);
        const int team = (int)threadIdx.x / items, item = (int)threadIdx.x % items;
        const int c = item / (D / 4), d = 4 * (item % (D / 4));
        float *mine = meet + (team * rows + c) * ROW;
        if (team < teams) {
            Kv4Sum z;
            for (int w0 = J.w_first + team; w0 <= J.w_last; w0 += 4 * teams) {
                float v[4][6];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int w = min(w0 + k * teams, J.w_last);
                    const float *src = A.part + ((int64_t)(2 * w + (w == J.w_first)) * KA_ROWS + c) * ROW;
#pragma unroll
                    for (int x = 0; x < 6; ++x)
                        v[k][x] = __hip_atomic_load(src + (x < 4 ? d + x : D + x - 4), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (w0 + k * teams <= J.w_last)
                        z.add(glint_f32x4{v[k][0], v[k][1], v[k][2], v[k][3]}, v[k][4], v[k][5]);
            }
            if (teams == 1) {
                z.store(kv4_out<D>(A, J.q0, J.h, J.rb * KA_ROWS + c) + d);
            } else {
                *(glint_f32x4 *)(mine + d) = z.o;
                if (d == 0) {
                    mine[D] = z.m;
                    mine[D + 1] = z.l;
                }
            }
        }
        if (teams > 1) {
            __syncthreads();
            if (team == 0) {
                Kv4Sum z;
                for (int t = 0; t < teams; ++t)
                    z.m = fmaxf(z.m, meet[(t * rows + c) * ROW + D]);
                for (int t = 0; t < teams; ++t) {
                    const float *from = meet + (t * rows + c) * ROW;
                    z.add_below(*(const glint_f32x4 *)(from + d), from[D], from[D + 1]);
                }
                z.store(kv4_out<D>(A, J.q0, J.h, J.rb * KA_ROWS + c) + d);
            }
            __syncthreads(); /* before the other group's teams write */
        }
        if (threadIdx.x == 0)
            __hip_atomic_store(&A.ctr[J.w_first], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

static bool ka_shape(int B, int max_q, int Hq, int H, int D, int max_pages) {
    return B >= 0 && max_q >= 1 && H >= 1 && Hq >= H && Hq % H == 0 && (D == 64 || D == 128) && max_pages >= 1 &&
           max_pages <= KA_FAR && (int64_t)max_q * (Hq / H) <= (1 << 20);
}

/* Groups that the shape allows a sequence, and how many sequences a launch takes so that all units of
 * cost fit 30 bits (0: not even one). */
static int64_t ka_groups(int max_q, int H, int G, int max_pages, int64_t &most) {
    const int64_t groups = ((int64_t)max_q * G + KA_ROWS - 1) / KA_ROWS * H;
    const int64_t units = (int64_t)max_pages + KA_WAVES + KA_SWITCH;
    most = groups > (1 << 30) / units ? 0 : (1 << 30) / (groups * units);
    return groups;
}

bool glint_serve_ws(hipStream_t stream, GlintSplitWs &ws) { return glint_split_ws_stream(stream, ws); }

GLINT_API int glint_serve_workspace_reserve(struct ihipStream_t *stream) {
    if (glint_stream_captures(stream))
        return -1;
    GlintSplitWs ws;
    return glint_serve_ws(stream, ws) ? 0 : -1;
}
GLINT_API int glint_serve_workspace_release(struct ihipStream_t *stream) { return glint_split_ws_release(stream); }

static int ka_attend(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq,
                               const uint8_t *k_hole, const float *k_absmax, const uint8_t *v_hole,
                               const float *v_absmax, int64_t pages, const int32_t *table, int64_t table_stride,
                               int max_pages, const int32_t *lens, const int32_t *cu_q, int B, int max_q, int Hq, int H,
                               int D, float scale, int window, int sinks, uint16_t *out, hipStream_t stream) {
    if (!q || !k_hole || !k_absmax || !v_hole || !v_absmax || !table || !lens || !out)
        return -1;
    if (!ka_shape(B, max_q, Hq, H, D, max_pages) || Tq < 0 || Tq > INT32_MAX || pages < 1 || pages >= (int64_t)1 << 40 ||
        (!cu_q && Tq != (int64_t)B * max_q) || window < 0 || window > GLINT_WINDOW_MAX || sinks < 0)
        return -2;
    if (!glint_aligned(q, 16) || !glint_aligned(out, 8) || !glint_aligned(k_hole, 16) || !glint_aligned(v_hole, 16) ||
        !glint_aligned(k_absmax, 16) || !glint_aligned(v_absmax, 16) || ((q_stride_t | q_stride_h) & 7))
        return -2;
    if (B == 0 || Tq == 0)
        return 0;
    const float scale2 = fabsf(scale) * (1.44269504088896341f / KV4_ALPHA);
    Kv4AttendArgs a{q, q_stride_t, q_stride_h, Tq, k_hole, v_hole, k_absmax, v_absmax, pages, table, table_stride,
                    max_pages, lens, cu_q, B, max_q, Hq, H, Hq / H, scale2 < FLT_MIN ? FLT_MIN : scale2,
                    scale < 0.f ? 0x80008000u : 0u, out, nullptr, nullptr, window, sinks};
    int64_t most;
    const int64_t groups = ka_groups(max_q, H, a.G, max_pages, most), cus = glint_cu_count();
    if (most < 1)
        return -2;
    GlintSplitWs ws;
    if (glint_serve_ws(stream, ws) && ws.nctr >= (size_t)cus &&
        ws.part_floats >= (size_t)cus * 2 * KA_ROWS * (D + 4)) {
        a.part = ws.part;
        a.ctr = ws.ctr;
    } else if (groups > INT32_MAX / KA_T) { /* a workgroup per group */
        return -2;
    } else {
        most = std::min<int64_t>(most, INT32_MAX / KA_T / groups);
    }
    for (int64_t b = 0; b < B; b += most) {
        a.B = (int)std::min<int64_t>(B - b, most);
        a.table = table + b * table_stride;
        a.lens = lens + b;
        if (cu_q) {
            a.cu_q = cu_q + b;
        } else { /* rows by number: this launch's alone */
            a.q = q + b * max_q * q_stride_t;
            a.out = out + b * max_q * Hq * D;
            a.Tq = (int64_t)a.B * max_q;
        }
        int64_t grid = a.B * groups;
        if (a.part)
            grid = std::min<int64_t>((grid * (max_pages + KA_WAVES + KA_SWITCH) + KA_WAVES - 1) / KA_WAVES, cus);
        const unsigned g = (unsigned)grid;
        if (D == 64 && !window)
            k_kv4_attend<64, false><<<g, KA_T, 0, stream>>>(a);
        else if (!window)
            k_kv4_attend<128, false><<<g, KA_T, 0, stream>>>(a);
        else if (D == 64)
            k_kv4_attend<64, true><<<g, KA_T, 0, stream>>>(a);
        else
            k_kv4_attend<128, true><<<g, KA_T, 0, stream>>>(a);
        if (hipGetLastError() != hipSuccess)
            return -3;
    }
    return 0;
}

GLINT_API int glint_kv4_attend(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq,
                               const uint8_t *k_hole, const float *k_absmax, const uint8_t *v_hole,
                               const float *v_absmax, int64_t pages, const int32_t *table, int64_t table_stride,
                               int max_pages, const int32_t *lens, const int32_t *cu_q, int B, int max_q, int Hq, int H,
                               int D, float scale, uint16_t *out, struct ihipStream_t *stream) {
    return ka_attend(q, q_stride_t, q_stride_h, Tq, k_hole, k_absmax, v_hole, v_absmax, pages, table, table_stride, max_pages,
                     lens, cu_q, B, max_q, Hq, H, D, scale, 0, 0, out, stream);
}

GLINT_API int glint_kv4_attend_window(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq,
                               const uint8_t *k_hole, const float *k_absmax, const uint8_t *v_hole,
                               const float *v_absmax, int64_t pages, const int32_t *table, int64_t table_stride,
                               int max_pages, const int32_t *lens, const int32_t *cu_q, int B, int max_q, int Hq, int H,
                               int D, float scale, int window, int sinks, uint16_t *out, struct ihipStream_t *stream) {
    return ka_attend(q, q_stride_t, q_stride_h, Tq, k_hole, k_absmax, v_hole, v_absmax, pages, table, table_stride, max_pages,
                     lens, cu_q, B, max_q, Hq, H, D, scale, window, sinks, out, stream);
}
