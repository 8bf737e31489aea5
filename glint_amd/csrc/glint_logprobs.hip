/* Log probabilities of given tokens (include/glint_serve.h).
 *
 * k_token_logprobs — one workgroup per row, one pass: a thread keeps a running maximum m,
 *   s = sum e^(x - m) and t = sum e^(x - m) (x - m) of its elements x, counts those that come
 *   before the token, and remembers the 16-B load that held its largest element. Then
 *     lse = m + ln s,  entropy = ln s - t / s.
 *   m is subtracted before the factor log2 e of the hardware's 2^x is applied: x log2 e
 *   overflows for the largest finite logits, which masks are made of.
 *   The top list needs no second pass over the row: with T the top-th largest of the threads'
 *   own maxima, every entry of the list is at least T and sits in one of the `top` threads
 *   whose maximum is at least T, so those threads look at their elements again and put
 *   what reaches T into LDS, at most top * (elements of a thread). Entries are compared as
 *   one 64-bit key, the value's order over the inverted index, so ties need no rule.
 *   Few long rows are split over workgroups, whose sums and lists meet in the last to arrive.
 *
 *   Long rows are bound by reading them once and, close behind, by some 14 vector instructions an
 *   element: 2047 rows of 128256 BF16 in 115 us, 4.6 TB/s, where a copy reaches 5.1, the vector units
 *   90% busy (m in powers of two saved 1 of them, 3 us, and overflowed); a second pass for the list
 *   would add to both. Short calls are bound by one chain of a
 *   workgroup's waits: first loads, wave and workgroup sums, the floor of the list, its
 *   candidates, their order; 8 rows of 128256 13 us. 1024 threads a row keep 64 KB of loads in
 *   flight; LP_U loads a thread and as many ahead. */
#include <algorithm>

#include "glint_common.h"
#include "glint_serve.h"
#include "serve_ws.h"

#define LP_T 1024
#define LP_WAVES (LP_T / 64)
#define LP_TOP 20
#define LP_T_MAX 0x3FFFFF /* rows of one launch */
#define LP_V_TOP 262144 /* longest row with a top list: its candidates fit LDS */
#define LP_SPLIT 32 /* most parts of a row */
#define LP_PART (4 + 2 * LP_TOP) /* words of a part: three sums, the count, the list */
/* a thread's 16-B loads hold at most LP_V_TOP / LP_T elements, rounded up to a load, and it
 * may own one element before and one after the aligned part */
#define LP_CAND (LP_TOP * (LP_V_TOP / LP_T + 8 + 2))

template <class E>
struct LpRow {
    static constexpr int PER = 16 / sizeof(E);
    const E *x;
    int64_t V;
    int head;     /* elements before the first 16-B boundary */
    int64_t nvec; /* 16-B loads */
    __device__ LpRow(const E *p, int64_t v) : x(p), V(v) {
        head = (int)min(v, (int64_t)((0u - (uint32_t)(uintptr_t)p) & 15u) / (int64_t)sizeof(E));
        nvec = (v - head) / PER;
    }
    __device__ float at(int64_t j) const;
    __device__ glint_u32x4 raw(int vec) const { return *(const glint_u32x4 *)(x + head + (int64_t)vec * PER); }
    __device__ void unpack(const glint_u32x4 u, float (&w)[PER]) const;
    /* the element of this thread's that lies outside the 16-B loads: before (thread j < head)
     * and after them, or -1 */
    __device__ int64_t before() const { return (int)threadIdx.x < head ? (int64_t)threadIdx.x : -1; }
    __device__ int64_t after() const {
        const int64_t j = head + nvec * PER + threadIdx.x;
        return j < V ? j : -1;
    }
};
template <>
__device__ __forceinline__ float LpRow<float>::at(int64_t j) const { return x[j]; }
template <>
__device__ __forceinline__ float LpRow<uint16_t>::at(int64_t j) const { return __uint_as_float((uint32_t)x[j] << 16); }
template <>
__device__ __forceinline__ void LpRow<float>::unpack(const glint_u32x4 u, float (&w)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = __uint_as_float(u[i]);
}
template <>
__device__ __forceinline__ void LpRow<uint16_t>::unpack(const glint_u32x4 u, float (&w)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[2 * i] = glint_bf16lo(u[i]);
        w[2 * i + 1] = glint_bf16hi(u[i]);
    }
}

/* Larger value, then lower index, is the larger key; NaN counts as -inf. Never 0. */
__device__ __forceinline__ uint64_t lp_key(float x, int64_t j) {
    uint32_t u = __float_as_uint(x != x ? -INFINITY : x + 0.f); /* + 0: -0 equals 0 */
    u = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return (uint64_t)u << 32 | (0xFFFFFFFFu - (uint32_t)j);
}
__device__ __forceinline__ uint32_t lp_key_index(uint64_t k) { return 0xFFFFFFFFu - (uint32_t)k; }
__device__ __forceinline__ float lp_key_value(uint64_t k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~u);
}
/* The next float above x; NaN above +inf and NaN. */
__device__ __forceinline__ float lp_next_up(float x) {
    const float y = x + 0.f;
    const int32_t i = __float_as_int(y);
    return y != y ? y : __int_as_float(i >= 0 ? i + 1 : i - 1);
}

/* Running sums of a set of elements: with a reference m (not below any x by more than LP_SLACK),
 * s = sum e^(x - m), t = sum e^(x - m) (x - m). */
#define LP_LOG2E 1.44269504088896341f
#define LP_SLACK 14.f
#define LP_FAR -1024.f /* e to this is 0, and a sum times it is finite: 0 times what lies farther counts 0 */
__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * LP_LOG2E); }
struct LpSum {
    float m, s, t;
    __device__ void shift(float to) { /* to > m */
        if (m != -INFINITY) {
            const float d = fmaxf(m - to, LP_FAR), f = lp_exp(d);
            t = f * fmaf(d, s, t);
            s = f * s;
        }
        m = to;
    }
    __device__ void add(float x) { /* m is finite, or x makes s NaN */
        const float d = x - m, e = lp_exp(d);
        s += e;
        t = fmaf(e, fmaxf(d, LP_FAR), t);
    }
};
/* Over each row of 16 lanes, left in every lane of the row. */
template <class F>
__device__ __forceinline__ float lp_row16(float v, F op) {
    v = op(v, __int_as_float(glint_dpp<GLINT_DPP_QUAD_1032>(__float_as_int(v))));
    v = op(v, __int_as_float(glint_dpp<GLINT_DPP_QUAD_2301>(__float_as_int(v))));
    v = op(v, __int_as_float(glint_dpp<GLINT_DPP_ROW_HALF_MIRROR>(__float_as_int(v))));
    return op(v, __int_as_float(glint_dpp<GLINT_DPP_ROW_MIRROR>(__float_as_int(v))));
}
__device__ __forceinline__ int lp_row16_sum(int v) {
    v += glint_dpp<GLINT_DPP_QUAD_1032>(v);
    v += glint_dpp<GLINT_DPP_QUAD_2301>(v);
    v += glint_dpp<GLINT_DPP_ROW_HALF_MIRROR>(v);
    return v + glint_dpp<GLINT_DPP_ROW_MIRROR>(v);
}
__device__ __forceinline__ float lp_lane(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
/* Over the wave: the four rows. The reads of other lanes stand here, in code that every lane
 * runs: a sum that only a branch uses may be computed inside it, for the branch's lanes alone. */
template <class F>
__device__ __forceinline__ float lp_wave(float v, F op) {
    v = lp_row16(v, op);
    return op(op(lp_lane(v, 0), lp_lane(v, 16)), op(lp_lane(v, 32), lp_lane(v, 48)));
}
__device__ __forceinline__ int lp_wave_sum(int v) {
    v = lp_row16_sum(v);
    return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
           __builtin_amdgcn_readlane(v, 48);
}
struct LpMax {
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct LpAdd {
    __device__ float operator()(float a, float b) const { return a + b; }
};
/* The sums under another reference `to` >= m; nothing but NaN is left of a set without one. */
__device__ __forceinline__ void lp_refer(LpSum &a, float to) {
    const float d = fmaxf(a.m - to, LP_FAR), f = a.m == -INFINITY ? 0.f : lp_exp(d);
    a.t = a.m == -INFINITY ? 0.f : f * fmaf(d, a.s, a.t);
    a.s = a.m == -INFINITY && a.s == a.s ? 0.f : f * a.s;
    a.m = to;
}

/* Largest of the wave's keys, in every lane: the upper words' maximum by DPP, then, where more
 * than one lane has it, the lower words'. */
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lp_dpp_max(uint32_t v) {
    const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
    return w > v ? w : v;
}
__device__ __forceinline__ uint32_t lp_wave_max32(uint32_t v) {
    v = lp_dpp_max<0x111, 0xF>(v); /* row_shr 1, 2, 4, 8 */
    v = lp_dpp_max<0x112, 0xF>(v);
    v = lp_dpp_max<0x114, 0xF>(v);
    v = lp_dpp_max<0x118, 0xF>(v);
    v = lp_dpp_max<0x142, 0xA>(v); /* row_bcast 15, 31 */
    v = lp_dpp_max<0x143, 0xC>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint64_t lp_wave_max(uint64_t v) {
    const uint32_t hi = lp_wave_max32((uint32_t)(v >> 32));
    const bool has = (uint32_t)(v >> 32) == hi;
    const uint64_t who = __ballot(has);
    uint32_t lo;
    if ((who & (who - 1)) == 0)
        lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, __builtin_ctzll(who));
    else
        lo = lp_wave_max32(has ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
}

/* A row's or a part's sums, and how many of its entries come before the token. */
struct LpPart {
    LpSum z;
    int n;
};
/* A row's outputs from its sums; `ref` and `ls` are what its top list needs. */
__device__ __forceinline__ void lp_write(const LpPart &p, int64_t tok, bool is_tok, float xt, bool writes, float *logprob,
                                         float *entropy, int32_t *rank, float &ref, float &log_sum) {
    const float s = p.z.m == -INFINITY ? NAN : p.z.s; /* nothing is possible */
    const float ls = logf(s);
    if (writes) {
        *logprob = tok < 0 ? 0.f : is_tok ? xt - p.z.m - ls : NAN;
        if (entropy)
            *entropy = ls - p.z.t / s;
        if (rank)
            *rank = is_tok ? p.n : -1;
        ref = p.z.m;
        log_sum = ls;
    }
}
/* How many of n keys are larger. */
__device__ __forceinline__ int lp_place(const uint64_t *keys, int n, uint64_t key) {
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i)
        place += keys[i] > key ? 1 : 0;
    return place;
}
/* The elements that reach `least` of every thread whose maximum does: the wave's lanes share those
 * threads' loads out, `rounds` of each thread. */
template <class E>
__device__ __forceinline__ void lp_candidates(const LpRow<E> &r, int v0, int nvec, int rounds, const int64_t (&ends)[2],
                                              uint64_t mine, uint64_t least, uint64_t *cand, int *ncand) {
    constexpr int PER = LpRow<E>::PER;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool has = mine != 0 && mine >= least;
    const uint64_t who = __ballot(has), below = who & ((1ull << lane) - 1);
    const int n = __builtin_popcountll(who), rank = __builtin_popcountll(below);
    /* lane i < n gets the i-th such thread's lane: every lane sends its own to a place of its own */
    const int order = __builtin_amdgcn_ds_permute(4 * (has ? rank : n + lane - rank), lane);
    for (int i0 = 0; i0 < n * rounds; i0 += 64) {
        const int i = i0 + lane, k = i % rounds;
        const int vec = wave * 64 + __shfl(order, min(i / rounds, 63), 64) + k * LP_T;
        if (i < n * rounds && vec < nvec) {
            float w[PER];
            r.unpack(r.raw(v0 + vec), w);
#pragma unroll
            for (int x = 0; x < PER; ++x) {
                const uint64_t key = lp_key(w[x], r.head + (int64_t)(v0 + vec) * PER + x);
                if (key >= least)
                    cand[atomicAdd(ncand, 1)] = key;
            }
        }
    }
    if (mine != 0 && mine >= least) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (ends[k] >= 0) {
                const uint64_t key = lp_key(r.at(ends[k]), ends[k]);
                if (key >= least)
                    cand[atomicAdd(ncand, 1)] = key;
            }
    }
}

#define LP_U 4 /* 16-B loads of a thread in flight, twice */

template <class E>
__global__ __launch_bounds__(LP_T, 8) void k_token_logprobs(const E *__restrict__ logits, int64_t stride,
                                                            const int64_t *__restrict__ tokens, int64_t V, int top,
                                                            float *__restrict__ logprob, float *__restrict__ entropy,
                                                            int32_t *__restrict__ rank, float *__restrict__ top_logprob,
                                                            int32_t *__restrict__ top_index, int nsplit, float *part,
                                                            unsigned *ctr) {
    constexpr int PER = LpRow<E>::PER;
    __shared__ float sm[LP_WAVES], ss[LP_WAVES], st[LP_WAVES];
    __shared__ int sr[LP_WAVES];
    __shared__ uint32_t wave_second[LP_WAVES];
    __shared__ uint64_t cand[LP_CAND];
    __shared__ uint64_t floor_key;
    __shared__ int ncand;
    __shared__ float s_ref, s_ls;
    __shared__ LpPart whole;
    __shared__ unsigned s_last;
    const int64_t row = blockIdx.x / nsplit;
    const int split = blockIdx.x % nsplit;
    const LpRow<E> r(logits + row * stride, V);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

    /* this workgroup's 16-B loads, v0 + threadIdx.x + k LP_T; one past the end repeats the last and
     * does not count */
    const int per = ((int)r.nvec + nsplit - 1) / nsplit, v0 = min(split * per, (int)r.nvec);
    const int nvec = min(per, (int)r.nvec - v0), rounds = (nvec + LP_T - 1) / LP_T;
    glint_u32x4 now[LP_U], next[LP_U];
    auto fetch = [&](int k0, glint_u32x4 (&w)[LP_U]) {
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
            w[u] = r.raw(v0 + min((int)threadIdx.x + (k0 + u) * LP_T, nvec - 1));
    };
    if (rounds > 0)
        fetch(0, now);

    const int64_t tok = tokens[row];
    const bool is_tok = tok >= 0 && tok < V;
    const float xt = is_tok ? r.at(tok) : NAN; /* NaN: nothing comes before it */
    /* entries that come before the token reach xt at indices below it and the next float above it */
    const float xt_up = lp_next_up(xt);

    LpSum a{-INFINITY, 0.f, 0.f};
    int before = 0;      /* this lane's ends */
    int wave_before = 0; /* the wave's loads, by ballots: every lane takes part in every round */
    float high = -INFINITY;
    int where = (int)threadIdx.x < nvec ? v0 + (int)threadIdx.x : -1;
    const uint32_t at = is_tok ? (uint32_t)tok : 0;
    auto take = [&](int vec, const glint_u32x4 raw) {
        float w[PER];
        r.unpack(raw, w);
        float mx = w[0];
#pragma unroll
        for (int i = 1; i < PER; ++i)
            mx = fmaxf(mx, w[i]);
        if (__any(mx - LP_SLACK > a.m)) {
            if (mx > a.m)
                a.shift(mx);
        }
        if (a.m != -INFINITY) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                a.add(w[i]);
        } else { /* nothing but -inf and NaN so far */
#pragma unroll
            for (int i = 0; i < PER; ++i)
                a.s += w[i] != w[i] ? NAN : 0.f;
        }
        const uint32_t j = (uint32_t)r.head + (uint32_t)vec * PER; /* V fits 31 bits; vec = -1: past every token */
        const float reach = j < at ? xt : xt_up;
        if (__any(mx >= reach)) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                wave_before += __builtin_popcountll(__ballot(w[i] >= reach));
            if (__any(j < at && at < j + PER)) { /* the token's own load: entries from it on that equal it */
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    wave_before -= __builtin_popcountll(__ballot(j < at && j + i >= at && w[i] == xt));
            }
        }
        where = mx > high ? vec : where;
        high = fmaxf(high, mx);
    };
    /* past the last load: -inf adds nothing, and at vec = -1 comes before no token, not even one at -inf */
    constexpr uint32_t NONE = sizeof(E) == 2 ? 0xFF80FF80u : 0xFF800000u;
    for (int k0 = 0; k0 < rounds; k0 += LP_U) {
        if (k0 + LP_U < rounds)
            fetch(k0 + LP_U, next);
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            if (k0 + u >= rounds)
                break;
            int vec = v0 + (int)threadIdx.x + (k0 + u) * LP_T;
            if ((k0 + u + 1) * LP_T > nvec) { /* the last round */
                const bool in = vec < v0 + nvec;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    now[u][i] = in ? now[u][i] : NONE;
                vec = in ? vec : -1;
            }
            take(vec, now[u]);
        }
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
            now[u] = next[u];
    }
    uint64_t mine = 0;
    const int64_t ends[2] = {split == 0 ? r.before() : -1, split == nsplit - 1 ? r.after() : -1};
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (ends[k] >= 0) {
            const float x = r.at(ends[k]);
            if (x > a.m)
                a.shift(x);
            if (a.m != -INFINITY)
                a.add(x);
            else
                a.s += x != x ? NAN : 0.f;
            before += x >= (ends[k] < tok ? xt : xt_up) ? 1 : 0;
            const uint64_t key = lp_key(x, ends[k]);
            mine = key > mine ? key : mine;
        }
    if (top > 0 && where >= 0) {
        float w[PER];
        r.unpack(r.raw(where), w);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint64_t key = lp_key(w[i], r.head + (int64_t)where * PER + i);
            mine = key > mine ? key : mine;
        }
    }
    /* the wave's sums under its largest reference */
    const float wm = lp_wave(a.m, LpMax());
    lp_refer(a, wm);
    const float ws = lp_wave(a.s, LpAdd()), wt = lp_wave(a.t, LpAdd());
    const int wr = lp_wave_sum(before) + wave_before;
    if (lane == 0) {
        sm[wave] = wm;
        ss[wave] = ws;
        st[wave] = wt;
        sr[wave] = wr;
    }
    /* A value that the top-th largest thread maximum is not below: two lanes of a wave reach the
     * second largest of its maxima, so where ceil(top / 2) waves reach a value by theirs, `top` lanes
     * do. The maxima that reach it, some 30 for a list of 20, count those before each of them: all 1024
     * where they are equal, as in a row of one value (8 such rows of 128256 33 us, 13 of others). */
    if (top > 0) {
        const uint32_t value = (uint32_t)(mine >> 32), first = lp_wave_max32(value);
        const bool is_first = value == first;
        const bool tie = __builtin_popcountll(__ballot(is_first)) > 1; /* every lane takes part */
        const uint32_t second = lp_wave_max32(is_first ? 0u : value);
        if (lane == 0)
            wave_second[wave] = tie ? first : second;
    }
    if (threadIdx.x == 0) {
        ncand = 0;
        floor_key = 0; /* fewer threads than `top` have an element: every element counts */
    }
    __syncthreads();
    if (wave == 0) {
        static_assert(LP_WAVES == 16, "one row of lanes holds every wave's sums");
        LpSum z{sm[lane & 15], ss[lane & 15], st[lane & 15]};
        const int n = lp_row16_sum(sr[lane & 15]);
        lp_refer(z, lp_row16(z.m, LpMax()));
        z.s = lp_row16(z.s, LpAdd());
        z.t = lp_row16(z.t, LpAdd());
        if (lane == 0)
            whole = LpPart{z, n};
    }
    if (top > 0) {
        const uint32_t own = wave_second[lane & 15];
        int ahead = 0; /* waves */
#pragma unroll
        for (int i = 0; i < LP_WAVES; ++i) {
            const uint32_t v = wave_second[i];
            ahead += v > own || (v == own && i < (lane & 15)) ? 1 : 0;
        }
        const uint64_t who = __ballot(ahead == (top - 1) / 2);
        const uint32_t reach = (uint32_t)__builtin_amdgcn_readlane((int)own, __builtin_ctzll(who));
        if (mine != 0 && (uint32_t)(mine >> 32) >= reach)
            cand[atomicAdd(&ncand, 1)] = mine;
        __syncthreads();
        const int n = ncand;
        for (int c = threadIdx.x; c < n; c += LP_T)
            if (lp_place(cand, n, cand[c]) == top - 1)
                floor_key = cand[c];
        __syncthreads();
        if (threadIdx.x == 0) { /* a list of one is that maximum */
            cand[0] = floor_key;
            ncand = top == 1 && floor_key != 0 ? 1 : 0;
        }
    }
    __syncthreads();
    if (nsplit == 1 && wave == 0)
        lp_write(whole, tok, is_tok, xt, lane == 0, logprob + row, entropy ? entropy + row : nullptr, rank ? rank + row : nullptr,
                 s_ref, s_ls);
    if (top > 1) {
        const uint64_t least = floor_key;
        lp_candidates(r, v0, nvec, rounds, ends, mine, least, cand, &ncand);
    }
    __syncthreads();
    if (nsplit > 1) {
        /* This part's sums and list go to the workspace; the part that arrives last takes all of
         * them as it took its threads': the largest of the lists' last entries is a floor. */
        uint32_t *mine_part = (uint32_t *)part + (row * nsplit + split) * LP_PART;
        if (threadIdx.x == 0) {
            const uint32_t v[4] = {__float_as_uint(whole.z.m), __float_as_uint(whole.z.s), __float_as_uint(whole.z.t),
                                   (uint32_t)whole.n};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                __hip_atomic_store(mine_part + i, v[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        auto put = [&](int place, uint64_t key) {
            __hip_atomic_store(mine_part + 4 + 2 * place, (uint32_t)key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(mine_part + 5 + 2 * place, (uint32_t)(key >> 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        const int n = top > 0 ? ncand : 0;
        for (int c = threadIdx.x; c < n; c += LP_T) {
            const int place = lp_place(cand, n, cand[c]);
            if (place < top)
                put(place, cand[c]);
        }
        if ((int)threadIdx.x < top && (int)threadIdx.x >= n)
            put(threadIdx.x, 0); /* a part shorter than the list */
        __builtin_amdgcn_s_waitcnt(GLINT_WAIT_VMCNT0);
        __syncthreads();
        if (threadIdx.x == 0) {
            s_last = __hip_atomic_fetch_add(ctr + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)nsplit - 1u;
            ncand = 0;
            floor_key = 0;
        }
        __syncthreads();
        if (!s_last)
            return;
        const uint32_t *parts = (const uint32_t *)part + row * nsplit * LP_PART;
        auto get = [&](int i) { return __hip_atomic_load(parts + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        auto key_of = [&](int p, int place) {
            return (uint64_t)get(p * LP_PART + 5 + 2 * place) << 32 | get(p * LP_PART + 4 + 2 * place);
        };
        const int p = (int)threadIdx.x / LP_TOP, place = (int)threadIdx.x % LP_TOP;
        const uint64_t key = p < nsplit && place < top ? key_of(p, place) : 0;
        if (wave == 0) {
            static_assert(LP_SPLIT <= 64, "a part a lane");
            LpPart z{{-INFINITY, 0.f, 0.f}, 0};
            uint64_t floor = 0;
            if (lane < nsplit) {
                z.z.m = __uint_as_float(get(lane * LP_PART));
                z.z.s = __uint_as_float(get(lane * LP_PART + 1));
                z.z.t = __uint_as_float(get(lane * LP_PART + 2));
                z.n = (int)get(lane * LP_PART + 3);
                floor = top > 0 ? key_of(lane, top - 1) : 0;
            }
            lp_refer(z.z, lp_wave(z.z.m, LpMax()));
            z.z.s = lp_wave(z.z.s, LpAdd());
            z.z.t = lp_wave(z.z.t, LpAdd());
            z.n = lp_wave_sum(z.n);
            lp_write(z, tok, is_tok, xt, lane == 0, logprob + row, entropy ? entropy + row : nullptr,
                     rank ? rank + row : nullptr, s_ref, s_ls);
            floor = lp_wave_max(floor);
            if (lane == 0) {
                floor_key = floor;
                __hip_atomic_store(ctr + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        __syncthreads();
        if (key != 0 && key >= floor_key)
            cand[atomicAdd(&ncand, 1)] = key;
        __syncthreads();
    }
    if (top == 0)
        return;
    const int n = ncand;
    const float m = s_ref, ls = s_ls;
    for (int c = threadIdx.x; c < n; c += LP_T) {
        const uint64_t key = cand[c];
        const int place = lp_place(cand, n, key);
        if (place < top) {
            top_logprob[row * top + place] = lp_key_value(key) - m - ls;
            top_index[row * top + place] = (int32_t)lp_key_index(key);
        }
    }
}

GLINT_API int glint_token_logprobs(const void *logits, int elt, int64_t stride, const int64_t *tokens, int64_t T,
                                   int64_t V, int top, float *logprob, float *entropy, int32_t *rank,
                                   float *top_logprob, int32_t *top_index, struct ihipStream_t *stream) {
    if (!logits || !tokens || !logprob || (top > 0 && (!top_logprob || !top_index)))
        return -1;
    if ((elt != GLINT_KV_BF16 && elt != GLINT_KV_F32) || T < 0 || T > LP_T_MAX || V < 1 || V > 0x7FFFFFFF || top < 0 ||
        top > LP_TOP || top > V || (top > 0 && V > LP_V_TOP) || !glint_aligned(logits, elt == GLINT_KV_BF16 ? 2 : 4))
        return -2;
    if (T == 0)
        return 0;
    /* Few rows are split, so that a workgroup per CU shares the reading, none with less than two loads
     * of every thread (as good as one, and fewer parts to join). Rows of 128256 BF16, split against
     * whole, by kernel: 8 rows with a list of 20 13.7 and 18.8 us, 64 without a list 9.8 and 15.7. */
    const int64_t parts = V / (elt == GLINT_KV_BF16 ? 8 : 4) / (2 * LP_T);
    int nsplit = (int)std::min<int64_t>(std::min<int64_t>(LP_SPLIT, parts), glint_cu_count() / T);
    GlintSplitWs ws{nullptr, nullptr, 0, 0};
    if (nsplit < 2 || !glint_serve_ws(stream, ws) || ws.nctr < (size_t)T ||
        ws.part_floats < (size_t)T * nsplit * LP_PART)
        nsplit = 1;
    const unsigned grid = (unsigned)T * nsplit;
    if (elt == GLINT_KV_BF16)
        k_token_logprobs<uint16_t><<<grid, LP_T, 0, stream>>>((const uint16_t *)logits, stride, tokens, V, top, logprob,
                                                              entropy, rank, top_logprob, top_index, nsplit, ws.part, ws.ctr);
    else
        k_token_logprobs<float><<<grid, LP_T, 0, stream>>>((const float *)logits, stride, tokens, V, top, logprob, entropy,
                                                           rank, top_logprob, top_index, nsplit, ws.part, ws.ctr);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
