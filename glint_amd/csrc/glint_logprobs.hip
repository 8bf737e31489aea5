/* Log probabilities of given tokens (include/glint_serve.h).
 *
 * k_token_logprobs — one workgroup per row, one pass: a thread keeps a running maximum m,
 *   s = sum e^(x - m) and t = sum e^(x - m) (x - m) of its elements, counts those that come
 *   before the token, and remembers the 16-B load that held its largest element. Then
 *     lse = m + log s,  entropy = log s - t / s.
 *   The top list needs no second pass over the row: with T the top-th largest of the threads'
 *   own maxima, every entry of the list is at least T and sits in one of the `top` threads
 *   whose maximum is at least T, so those threads look at their elements again and put
 *   what reaches T into LDS, at most top * (elements of a thread). Entries are compared as
 *   one 64-bit key, the value's order over the inverted index, so ties need no rule. */
#include "glint_common.h"
#include "glint_serve.h"

#define LP_T 1024
#define LP_WAVES (LP_T / 64)
#define LP_TOP 20
#define LP_T_MAX 0x3FFFFF /* rows of one launch */
#define LP_V_TOP 262144 /* longest row with a top list: its candidates fit LDS */
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
    __device__ void load(int64_t vec, float (&w)[PER]) const;
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
__device__ __forceinline__ void LpRow<float>::load(int64_t vec, float (&w)[4]) const {
    const glint_f32x4 u = *(const glint_f32x4 *)(x + head + vec * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = u[i];
}
template <>
__device__ __forceinline__ void LpRow<uint16_t>::load(int64_t vec, float (&w)[8]) const {
    const glint_u32x4 u = *(const glint_u32x4 *)(x + head + vec * 8);
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
__device__ __forceinline__ uint64_t lp_wave_max(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor(v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}

struct LpSum {
    float m, s, t;
    /* one more element; -inf adds nothing */
    __device__ void shift(float to) { /* to >= m */
        if (to > m) {
            if (m != -INFINITY) {
                const float d = m - to, f = __builtin_amdgcn_exp2f(d * 1.44269504088896341f);
                t = f * fmaf(d, s, t);
                s = f * s;
            }
            m = to;
        }
    }
    __device__ void add(float x) {
        const float d = x - m, e = __builtin_amdgcn_exp2f(d * 1.44269504088896341f);
        s += e;
        t = fmaf(e, x == -INFINITY ? 0.f : d, t);
    }
};
__device__ __forceinline__ void lp_join(LpSum &a, float m, float s, float t) {
    const float to = fmaxf(a.m, m);
    if (to == -INFINITY) {
        a.s += s; /* NaN stays NaN */
        return;
    }
    const float da = a.m - to, db = m - to;
    const float fa = __builtin_amdgcn_exp2f(da * 1.44269504088896341f), fb = __builtin_amdgcn_exp2f(db * 1.44269504088896341f);
    const float ta = a.m == -INFINITY ? a.t : fmaf(da, a.s, a.t), tb = m == -INFINITY ? t : fmaf(db, s, t);
    a.s = fmaf(fa, a.s, fb * s);
    a.t = fmaf(fa, ta, fb * tb);
    a.m = to;
}

template <class E>
__global__ __launch_bounds__(LP_T) void k_token_logprobs(const E *__restrict__ logits, int64_t stride,
                                                         const int64_t *__restrict__ tokens, int64_t V, int top,
                                                         float *__restrict__ logprob, float *__restrict__ entropy,
                                                         int32_t *__restrict__ rank, float *__restrict__ top_logprob,
                                                         int32_t *__restrict__ top_index) {
    constexpr int PER = LpRow<E>::PER;
    __shared__ float sm[LP_WAVES], ss[LP_WAVES], st[LP_WAVES];
    __shared__ int sr[LP_WAVES];
    __shared__ uint64_t best[LP_WAVES * LP_TOP], cand[LP_CAND];
    __shared__ uint64_t floor_key;
    __shared__ int ncand;
    __shared__ float s_lse;
    const int64_t row = blockIdx.x;
    const LpRow<E> r(logits + row * stride, V);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tok = tokens[row];
    const bool is_tok = tok >= 0 && tok < V;
    const float xt = is_tok ? r.at(tok) : INFINITY;

    LpSum a{-INFINITY, 0.f, 0.f};
    int before = 0;
    uint64_t mine = 0;
    float high = -INFINITY;
    int64_t where = -1;
    bool bad = false; /* NaN or +inf */
    for (int64_t vec = threadIdx.x; vec < r.nvec; vec += LP_T) {
        float w[PER];
        r.load(vec, w);
        float mx = w[0];
#pragma unroll
        for (int i = 1; i < PER; ++i)
            mx = fmaxf(mx, w[i]);
        a.shift(mx);
        if (a.m != -INFINITY) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                a.add(w[i]);
        }
        const int64_t j = r.head + vec * PER;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            before += w[i] > xt || (w[i] == xt && j + i < tok) ? 1 : 0;
            bad |= !(w[i] < INFINITY);
        }
        if (mx > high || where < 0) {
            high = fmaxf(high, mx); /* not NaN */
            where = vec;
        }
    }
    int64_t ends[2] = {r.before(), r.after()};
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (ends[k] >= 0) {
            const float x = r.at(ends[k]);
            a.shift(x);
            if (a.m != -INFINITY)
                a.add(x);
            before += x > xt || (x == xt && ends[k] < tok) ? 1 : 0;
            bad |= !(x < INFINITY);
            const uint64_t key = lp_key(x, ends[k]);
            mine = key > mine ? key : mine;
        }
    if (top > 0 && where >= 0) {
        float w[PER];
        r.load(where, w);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint64_t key = lp_key(w[i], r.head + where * PER + i);
            mine = key > mine ? key : mine;
        }
    }
    if (bad)
        a.s = NAN;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lp_join(a, __shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.t, o, 64));
        before += __shfl_xor(before, o, 64);
    }
    if (lane == 0) {
        sm[wave] = a.m;
        ss[wave] = a.s;
        st[wave] = a.t;
        sr[wave] = before;
    }
    /* this wave's `top` largest thread maxima, in order */
    uint64_t rest = mine;
    for (int i = 0; i < top; ++i) {
        const uint64_t k = lp_wave_max(rest);
        if (lane == 0)
            best[wave * LP_TOP + i] = k;
        if (rest == k)
            rest = 0; /* keys differ, but for 0 */
    }
    if (threadIdx.x == 0)
        ncand = 0;
    __syncthreads();
    if (wave == 0) {
        LpSum z{-INFINITY, 0.f, 0.f};
        int n = 0;
        for (int i = 0; i < LP_WAVES; ++i) {
            lp_join(z, sm[i], ss[i], st[i]);
            n += sr[i];
        }
        if (z.m == -INFINITY)
            z.s = NAN; /* nothing is possible */
        const float ls = logf(z.s);
        const float lse = z.m + ls;
        if (lane == 0) {
            logprob[row] = tok < 0 ? 0.f : is_tok ? (xt - z.m) - ls : NAN;
            if (entropy)
                entropy[row] = ls - z.t / z.s;
            if (rank)
                rank[row] = is_tok ? n : -1;
            s_lse = lse;
        }
        /* the top-th largest over the waves */
        uint64_t v[(LP_WAVES * LP_TOP + 63) / 64];
#pragma unroll
        for (int i = 0; i < (LP_WAVES * LP_TOP + 63) / 64; ++i) {
            const int k = lane + 64 * i;
            v[i] = k < LP_WAVES * LP_TOP && k % LP_TOP < top ? best[k] : 0;
        }
        uint64_t k = 0;
        for (int i = 0; i < top; ++i) {
            k = 0;
#pragma unroll
            for (int u = 0; u < (LP_WAVES * LP_TOP + 63) / 64; ++u)
                k = v[u] > k ? v[u] : k;
            k = lp_wave_max(k);
#pragma unroll
            for (int u = 0; u < (LP_WAVES * LP_TOP + 63) / 64; ++u)
                v[u] = v[u] == k ? 0 : v[u];
        }
        if (lane == 0)
            floor_key = k;
    }
    if (top == 0)
        return;
    __syncthreads();
    const uint64_t least = floor_key;
    if (mine != 0 && mine >= least) {
        for (int64_t vec = threadIdx.x; vec < r.nvec; vec += LP_T) {
            float w[PER];
            r.load(vec, w);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint64_t key = lp_key(w[i], r.head + vec * PER + i);
                if (key >= least)
                    cand[atomicAdd(&ncand, 1)] = key;
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (ends[k] >= 0) {
                const uint64_t key = lp_key(r.at(ends[k]), ends[k]);
                if (key >= least)
                    cand[atomicAdd(&ncand, 1)] = key;
            }
    }
    __syncthreads();
    const int n = ncand;
    const float lse = s_lse;
    for (int c = threadIdx.x; c < n; c += LP_T) {
        const uint64_t key = cand[c];
        int place = 0;
        for (int i = 0; i < n; ++i)
            place += cand[i] > key ? 1 : 0;
        if (place < top) {
            const uint32_t j = lp_key_index(key);
            top_logprob[row * top + place] = r.at(j) - lse;
            top_index[row * top + place] = (int32_t)j;
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
    if (elt == GLINT_KV_BF16)
        k_token_logprobs<uint16_t><<<(unsigned)T, LP_T, 0, stream>>>((const uint16_t *)logits, stride, tokens, V, top,
                                                                     logprob, entropy, rank, top_logprob, top_index);
    else
        k_token_logprobs<float><<<(unsigned)T, LP_T, 0, stream>>>((const float *)logits, stride, tokens, V, top,
                                                                  logprob, entropy, rank, top_logprob, top_index);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
