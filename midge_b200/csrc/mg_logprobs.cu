// mg_logprobs.cu -- log probabilities of given tokens, the entropy of the
// distribution and its top alternatives, per logits row x of V entries:
//   z = log sum e^(x_i - m),  m = max x
//   log p_i = (x_i - m) - z,  H = z - sum e^(x_i - m) (x_i - m) / sum e^(x_i - m)
//
// One pass over the row, 16 bytes a thread at a time: a running maximum, sum
// and weighted sum per thread (fp32, rescaled when the maximum moves), joined
// at the end.  The alternatives need no second pass: every thread knows its
// own maximum, the k-th largest of the block's 64 group maxima is a lower
// bound of the k-th largest entry, and only the threads whose maximum reaches
// it (a few more than k) have entries to collect again, from L2; the handful
// of candidates is ranked by counting.  A call of few rows cuts each row over
// several blocks and the last one to finish joins them, in block order.
// Bound: HBM (one read of the logits).  Measured: 2047 rows of 151936 bf16, 20
// alternatives: 138 us (622 MB, 4.5 TB/s); what is missing is each row's end
// (joins and ranking, some 3 us with three blocks an SM to cover it) and the
// exponentials.  8 rows of 201088 f32, 5 alternatives: 11 us, a launch, one
// round of loads and the join of the row's pieces.  Rows that are nearly all
// one number (masked by the lowest one, fewer tokens left than alternatives)
// have more candidates than fit and take a pass per alternative: 13 ms for
// the first of these cases.  Sums are fp32, exponentials ex2.approx: within
// 1e-7 of a log probability's size.
#include <string.h>

#include <type_traits>

#include "mg_kv4.cuh"

namespace mg {

constexpr int LP_THREADS = 512;
constexpr int LP_GROUPS = 64, LP_LANES = LP_THREADS / LP_GROUPS;  // groups of 8 lanes, one maximum each
// Candidates that fit shared memory: whole rows of up to 2048 entries, since 16-bit rows below that have their vectors in
// fewer groups than there may be alternatives, so that every entry is one (2048 rows of 1500, 32 alternatives: 294 us with
// room for 1024)
constexpr int LP_CAND = 2048;
constexpr int LP_UNROLL = 4;                                      // 16-byte loads of a thread in flight
constexpr int LP_MAX_PARTS = 1024, LP_MAX_ROWS = 512;             // of a call that cuts rows
constexpr float LP_LOG2E = 1.4426950408889634f;
static_assert(MG_LOGPROBS_MAX_ALT <= LP_GROUPS, "the bound takes a maximum per alternative");

struct LpPart {  // of one piece of a row: statistics, and its best entries in order (id -1: none)
    float m, s, w, pad;
    float v[MG_LOGPROBS_MAX_ALT];
    int32_t id[MG_LOGPROBS_MAX_ALT];
};

struct LpArgs {
    const void *x;
    int64_t ldx, V;
    int n_rows, n_ids, top, splits;
    const int32_t *ids;
    float *lp, *entropy, *top_lp;
    int32_t *top_ids;
    unsigned *count;  // [n_rows], of cut rows
    LpPart *parts;    // [n_rows][splits]
};

struct LpSmem {
    float gmax[LP_GROUPS];
    float red[3][LP_THREADS / 32];
    float cv[LP_CAND];
    int32_t ci[LP_CAND];
    uint16_t who[LP_THREADS];  // threads whose maximum reaches the bound
    float bound;
    int n, nwho, last;
    int kept;  // candidates that lp_thin keeps: not n, which other warps may still be reading when it starts
};

__device__ __forceinline__ float lp_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ bool better(float v, int32_t i, float w, int32_t j) { return v > w || (v == w && i < j); }
// NaN counts as -infinity
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }

// Sum and weighted sum against a maximum m, moved to the maximum M >= m.  Where nothing is left of them (87 or more
// apart, m = -infinity among these) they are 0: s times such a d may pass fp32.
__device__ __forceinline__ void lp_move(float &s, float &w, float m, float M) {
    const float d = fmaxf(m - M, -1e30f), f = lp_ex2(d * LP_LOG2E);
    w = f > 0.f ? f * (w + s * d) : 0.f;
    s = f > 0.f ? f * s : 0.f;
}

// A thread's sums are against a reference r that follows its maximum m only when that is LP_AHEAD above it (e^40 times the
// entries stays far inside fp32): a running maximum moves in some lane of a warp nearly every time.
constexpr float LP_AHEAD = 40.f;
struct LpAcc {
    float m = -INFINITY, r = -INFINITY, s = 0.f, w = 0.f;
    // entries one after another, -infinity (and NaN, made so) among them
    template <int N>
    __device__ __forceinline__ void add_any(const float (&v)[N]) {
        const float rr = r == -INFINITY ? 0.f : r;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float d = fmaxf(v[i] - rr, -1e30f), e = lp_ex2(d * LP_LOG2E);
            s += e;
            w = fmaf(e, d, w);
        }
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N]) {
        float top = m;
#pragma unroll
        for (int i = 0; i + 1 < N; i += 2) top = max3(top, v[i], v[i + 1]);
        if (N & 1) top = fmaxf(top, v[N - 1]);
        m = top;
        if (top > r + LP_AHEAD) {  // r = -infinity: any number
            lp_move(s, w, r, top);
            r = top;
        }
        if constexpr (N % 2 == 0) {
            float2 es = make_float2(0.f, 0.f), ws = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float2 d = add2(make_float2(v[i], v[i + 1]), make_float2(-r, -r));
                const float2 t = mul2(d, make_float2(LP_LOG2E, LP_LOG2E));
                const float2 e = make_float2(lp_ex2(t.x), lp_ex2(t.y));
                es = add2(es, e);
                ws = fma2(e, d, ws);
            }
            const float wx = ws.x + ws.y;
            if (wx == wx) {  // a -infinity or NaN entry (or nothing else yet) makes it NaN
                s += es.x + es.y;
                w += wx;
                return;
            }
        }
        add_any(v);
    }
};

// The row's piece [a, b): a scalar head up to 16-byte alignment, 16-byte
// vectors, a scalar tail.  Thread t has vectors t, t + LP_THREADS, ...; the
// head and tail belong to the first threads.
template <typename T>
struct LpSpan {
    static constexpr int E = 16 / sizeof(T);
    const T *x;
    int64_t a, b, va;  // va: first entry of the vectors
    int nv, nhead, ntail;
    __device__ __forceinline__ LpSpan(const T *row, int64_t a_, int64_t b_) : x(row), a(a_), b(b_) {
        const int64_t mis = (reinterpret_cast<uintptr_t>(row + a) & 15) / sizeof(T);
        nhead = (int)(mis ? min((int64_t)E - mis, b - a) : 0);
        va = a + nhead;
        nv = (int)((b - va) / E);
        ntail = (int)(b - va - (int64_t)nv * E);
    }
    // thread t's scalar entry, or -1
    __device__ __forceinline__ int64_t edge(int t) const {
        return t < nhead ? a + t : (t < nhead + ntail ? b - ntail + (t - nhead) : -1);
    }
    __device__ __forceinline__ uint4 vec(int i) const { return __ldg(reinterpret_cast<const uint4 *>(x + va) + i); }
    static __device__ __forceinline__ void unpack(const uint4 &q, float *v) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // an operation an entry
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
            T e[E];
            memcpy(e, &q, 16);
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = to_f32(e[i]);
        }
    }
};

// the top-th largest of the block's 64 group maxima (sm.gmax) into sm.bound, by two warps
__device__ __forceinline__ void lp_bound(LpSmem &sm, int top) {
    if (threadIdx.x >= LP_GROUPS) return;
    const float g = sm.gmax[threadIdx.x];
    int r = 0;
#pragma unroll 16
    for (int j = 0; j < LP_GROUPS; j++) {
        const float o = sm.gmax[j];
        r += o > g || (o == g && j < (int)threadIdx.x);
    }
    if (r == top - 1) sm.bound = g;
}

// The candidates thinned the way the row was, where there are more than
// ranking by counting is good for (short rows, whose entries few threads
// hold): each thread has n / LP_THREADS of them.  The block's threads
// together, with the same n: nothing here writes what n was read from.
constexpr int LP_MANY = 96;
__device__ __forceinline__ int lp_thin(LpSmem &sm, int n, int top) {
    if (n <= LP_MANY) return n;
    constexpr int K = LP_CAND / LP_THREADS;
    float v[K], g = -INFINITY;
    int32_t id[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int i = k * LP_THREADS + threadIdx.x;
        v[k] = i < n ? sm.cv[i] : -INFINITY;
        id[k] = i < n ? sm.ci[i] : -1;
        g = fmaxf(g, v[k]);
    }
#pragma unroll
    for (int o = LP_LANES / 2; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (threadIdx.x % LP_LANES == 0) sm.gmax[threadIdx.x / LP_LANES] = g;
    if (threadIdx.x == 0) sm.kept = 0;
    __syncthreads();
    lp_bound(sm, top);
    __syncthreads();
    const float bound = sm.bound;
#pragma unroll
    for (int k = 0; k < K; k++)
        if (id[k] >= 0 && v[k] >= bound) {
            const int c = atomicAdd(&sm.kept, 1);
            sm.cv[c] = v[k];
            sm.ci[c] = id[k];
        }
    __syncthreads();
    return sm.kept;
}

// With fewer than `top` possible tokens in [a, b) (n of them, ranked already)
// the next are the first banned ones (-infinity, NaN) by index: warp 0 looks
// for them from a on, and all but n entries are such.
template <typename T, typename F>
__device__ __forceinline__ void lp_banned(const T *x, int64_t a, int64_t b, int n, int top, F &&out) {
    if (threadIdx.x >= 32) return;
    int r = n;
    for (int64_t i0 = a; i0 < b && r < top; i0 += 32) {
        const int64_t i = i0 + threadIdx.x;
        const bool is = i < b && clean(to_f32(x[i])) == -INFINITY;
        const unsigned who = __ballot_sync(0xffffffffu, is);
        const int mine = r + __popc(who & ((1u << threadIdx.x) - 1u));
        if (is && mine < top) out(mine, -INFINITY, (int32_t)i);
        r += __popc(who);
    }
    for (r += threadIdx.x; r < top; r += 32) out(r, -INFINITY, -1);
}

// ranks the candidates sm.cv / sm.ci (n of them, distinct indexes) and calls out(rank, value, index) for the best `top`
template <typename F>
__device__ __forceinline__ void lp_rank(const LpSmem &sm, int n, int top, F &&out) {
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const float v = sm.cv[i];
        const int32_t id = sm.ci[i];
        int r = 0;
        for (int j = 0; j < n; j++) r += better(sm.cv[j], sm.ci[j], v, id);
        if (r < top) out(r, v, id);
    }
}

// the best `top` of [a, b) one after another, a pass for each: where the candidates do not fit (rows of equal entries,
// nearly everything banned)
template <typename T, typename F>
__device__ void lp_slow(const T *x, int64_t a, int64_t b, int top, LpSmem &sm, F &&out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float lv = INFINITY;
    int32_t li = -1;
    for (int r = 0; r < top; r++) {
        float v = -INFINITY;
        int32_t id = 0x7fffffff;
        for (int64_t i = a + threadIdx.x; i < b; i += LP_THREADS) {
            const float y = clean(to_f32(x[i]));
            if (better(lv, li, y, (int32_t)i) && better(y, (int32_t)i, v, id)) {
                v = y;
                id = (int32_t)i;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, v, o);
            const int32_t oi = __shfl_xor_sync(0xffffffffu, id, o);
            if (better(ov, oi, v, id)) { v = ov; id = oi; }
        }
        __syncthreads();
        if (lane == 0) { sm.cv[warp] = v; sm.ci[warp] = id; }
        __syncthreads();
        for (int k = 0; k < LP_THREADS / 32; k++)
            if (better(sm.cv[k], sm.ci[k], v, id)) { v = sm.cv[k]; id = sm.ci[k]; }
        lv = v;
        li = id;
        if (threadIdx.x == 0) out(r, v, id == 0x7fffffff ? -1 : id);
    }
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 3) k_logprobs(LpArgs a) {
    __shared__ LpSmem sm;
    constexpr int E = LpSpan<T>::E;
    const int row = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.ldx;
    const int64_t p0 = a.V * part / a.splits, p1 = a.V * (part + 1) / a.splits;
    const LpSpan<T> sp(x, p0, p1);
    if (tid == 0) sm.n = sm.nwho = 0;

    // ---- the pass
    LpAcc acc;
    {
        const int64_t i = sp.edge(tid);
        if (i >= 0) {
            const float v[1] = {clean(to_f32(x[i]))};
            acc.add(v);
        }
    }
    int i = tid;
    for (; i + (LP_UNROLL - 1) * LP_THREADS < sp.nv; i += LP_UNROLL * LP_THREADS) {
        uint4 q[LP_UNROLL];
#pragma unroll
        for (int k = 0; k < LP_UNROLL; k++) q[k] = sp.vec(i + k * LP_THREADS);
        constexpr int AT = 16 / E;  // vectors of 16 entries
#pragma unroll
        for (int k = 0; k < LP_UNROLL; k += AT) {
            float v[16];
#pragma unroll
            for (int j = 0; j < AT; j++) LpSpan<T>::unpack(q[k + j], v + j * E);
            acc.add(v);
        }
    }
    for (; i < sp.nv; i += LP_THREADS) {
        float v[E];
        LpSpan<T>::unpack(sp.vec(i), v);
        acc.add(v);
    }

    // ---- the block's statistics, and the groups' maxima
    float g = acc.m;
#pragma unroll
    for (int o = LP_LANES / 2; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % LP_LANES == 0) sm.gmax[tid / LP_LANES] = g;
    __syncthreads();
    const float M = warp_max(fmaxf(sm.gmax[lane], sm.gmax[lane + 32]));
    float s = acc.s, w = acc.w;
    lp_move(s, w, acc.r, M == -INFINITY ? 0.f : M);
    s = warp_sum(s);
    w = warp_sum(w);
    if (lane == 0) {
        sm.red[0][warp] = s;
        sm.red[1][warp] = w;
    }
    if (a.top > 0) lp_bound(sm, a.top);
    __syncthreads();
    s = w = 0.f;
#pragma unroll
    for (int k = 0; k < LP_THREADS / 32; k++) {
        s += sm.red[0][k];
        w += sm.red[1][k];
    }

    // ---- candidates: the entries that reach the bound, from the threads that have one
    if (a.top > 0) {
        const float bound = sm.bound;
        auto take = [&](float v, int64_t at) {
            if (v >= bound && v > -INFINITY) {
                const int k = atomicAdd(&sm.n, 1);
                if (k < LP_CAND) {
                    sm.cv[k] = v;
                    sm.ci[k] = (int32_t)at;
                }
            }
        };
        const int64_t ei = sp.edge(tid);
        if (ei >= 0) take(clean(to_f32(x[ei])), ei);
        if (acc.m >= bound) sm.who[atomicAdd(&sm.nwho, 1)] = (uint16_t)tid;
        __syncthreads();
        // their vectors, all at once over the block's threads
        const int each = (sp.nv + LP_THREADS - 1) / LP_THREADS, pairs = sm.nwho * each;
#pragma unroll 2
        for (int k = tid; k < pairs; k += LP_THREADS) {
            const int t = k / each, at = sm.who[t] + (k - t * each) * LP_THREADS;
            if (at >= sp.nv) continue;
            float v[E];
            LpSpan<T>::unpack(sp.vec(at), v);
#pragma unroll
            for (int e = 0; e < E; e++) take(clean(v[e]), sp.va + (int64_t)at * E + e);
        }
        __syncthreads();
    }
    int n = sm.n;
    if (a.top > 0 && n <= LP_CAND) n = lp_thin(sm, n, a.top);

    const float Mz = M == -INFINITY ? 0.f : M;
    if (a.splits == 1) {
        // no possible token: z = 0, so that every log probability is -infinity; +infinity among the logits: NaN
        const float z = M == INFINITY ? NAN : (s > 0.f ? logf(s) : 0.f);
        if (tid == 0) a.entropy[row] = s > 0.f ? z - w / s : z;
        for (int k = tid; k < a.n_ids; k += LP_THREADS) {
            const int32_t id = a.ids[(int64_t)row * a.n_ids + k];
            a.lp[(int64_t)row * a.n_ids + k] = id >= 0 && id < a.V ? clean(to_f32(x[id])) - Mz - z : 0.f;
        }
        auto out = [&](int r, float v, int32_t id) {
            a.top_ids[(int64_t)row * a.top + r] = id;
            a.top_lp[(int64_t)row * a.top + r] = id >= 0 ? v - Mz - z : -INFINITY;
        };
        if (a.top > 0) {
            if (n <= LP_CAND) {
                lp_rank(sm, n, a.top, out);
                if (n < a.top) lp_banned(x, p0, p1, n, a.top, out);
            } else {
                lp_slow(x, p0, p1, a.top, sm, out);
            }
        }
        return;
    }

    // ---- a piece of a row: its part, and the last block joins them
    LpPart *parts = a.parts + (size_t)row * a.splits, *mine = parts + part;
    if (tid == 0) {
        mine->m = M;
        mine->s = s;
        mine->w = w;
    }
    auto keep = [&](int r, float v, int32_t id) {
        mine->v[r] = v;
        mine->id[r] = id;
    };
    if (a.top > 0) {
        if (n <= LP_CAND) {
            lp_rank(sm, n, a.top, keep);
            for (int r = n + tid; r < a.top; r += LP_THREADS) keep(r, -INFINITY, -1);  // the join looks for banned ones
        } else {
            lp_slow(x, p0, p1, a.top, sm, keep);
        }
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        const bool last = atomicAdd(&a.count[row], 1u) + 1u == (unsigned)a.splits;
        if (last) a.count[row] = 0u;  // ready for the next call
        sm.last = last;
        sm.n = 0;
        __threadfence();
    }
    __syncthreads();
    if (!sm.last) return;
    // every warp joins the statistics, each lane some parts; the bound: the best of the parts' last entries
    float jm = -INFINITY, jb = -INFINITY;
    for (int k = lane; k < a.splits; k += 32) {
        jm = fmaxf(jm, __ldcg(&parts[k].m));
        if (a.top > 0) jb = fmaxf(jb, __ldcg(&parts[k].v[a.top - 1]));
    }
    jm = warp_max(jm);
    jb = warp_max(jb);
    const float jz = jm == -INFINITY ? 0.f : jm;
    float js = 0.f, jw = 0.f;
    for (int k = lane; k < a.splits; k += 32) {
        float ps = __ldcg(&parts[k].s), pw = __ldcg(&parts[k].w);
        lp_move(ps, pw, __ldcg(&parts[k].m), jz);
        js += ps;
        jw += pw;
    }
    js = warp_sum(js);
    jw = warp_sum(jw);
    const float z = jm == INFINITY ? NAN : (js > 0.f ? logf(js) : 0.f);
    if (tid == 0) a.entropy[row] = js > 0.f ? z - jw / js : z;
    for (int k = tid; k < a.n_ids; k += LP_THREADS) {
        const int32_t id = a.ids[(int64_t)row * a.n_ids + k];
        a.lp[(int64_t)row * a.n_ids + k] = id >= 0 && id < a.V ? clean(to_f32(x[id])) - jz - z : 0.f;
    }
    if (a.top == 0) return;
    for (int k = tid; k < a.splits * a.top; k += LP_THREADS) {
        const LpPart *p = parts + k / a.top;
        const float v = __ldcg(&p->v[k % a.top]);
        const int32_t id = __ldcg(&p->id[k % a.top]);
        if (id >= 0 && v >= jb && v > -INFINITY) {
            const int c = atomicAdd(&sm.n, 1);
            if (c < LP_CAND) {
                sm.cv[c] = v;
                sm.ci[c] = id;
            }
        }
    }
    __syncthreads();
    auto out = [&](int r, float v, int32_t id) {
        a.top_ids[(int64_t)row * a.top + r] = id;
        a.top_lp[(int64_t)row * a.top + r] = id >= 0 ? v - jz - z : -INFINITY;
    };
    int jn = sm.n;
    if (jn <= LP_CAND) jn = lp_thin(sm, jn, a.top);
    if (jn <= LP_CAND) {
        lp_rank(sm, jn, a.top, out);
        if (jn < a.top) lp_banned(x, 0, a.V, jn, a.top, out);
    } else {
        lp_slow(x, 0, a.V, a.top, sm, out);
    }
}

// Pieces of a row: what fills the GPU at three blocks an SM, of 4 vectors a
// thread at least.
template <typename T>
static int lp_splits(int64_t V, int n_rows) {
    int64_t s = (int64_t)num_sms() * 3 / n_rows;
    const int64_t most = V / ((int64_t)LP_THREADS * 4 * LpSpan<T>::E);
    if (s > most) s = most;
    if (s > LP_MAX_PARTS / n_rows) s = LP_MAX_PARTS / n_rows;
    return s < 1 || n_rows > LP_MAX_ROWS ? 1 : (int)s;
}

template <typename T>
static int logprobs_t(LpArgs &a, cudaStream_t st) {
    a.splits = lp_splits<T>(a.V, a.n_rows);
    // rows by the grid's y (65535 at most) a launch at a time
    for (int r = 0; r < a.n_rows; r += 65535) {
        LpArgs b = a;
        b.n_rows = a.n_rows - r < 65535 ? a.n_rows - r : 65535;
        b.x = static_cast<const T *>(a.x) + (int64_t)r * a.ldx;
        b.ids = a.ids ? a.ids + (int64_t)r * a.n_ids : nullptr;
        b.lp = a.lp ? a.lp + (int64_t)r * a.n_ids : nullptr;
        b.entropy = a.entropy + r;
        b.top_ids = a.top_ids ? a.top_ids + (int64_t)r * a.top : nullptr;
        b.top_lp = a.top_lp ? a.top_lp + (int64_t)r * a.top : nullptr;
        k_logprobs<T><<<dim3(b.splits, b.n_rows), LP_THREADS, 0, st>>>(b);
        MG_CHECK_LAUNCH();
    }
    return MG_OK;
}

}  // namespace mg

using namespace mg;

static int lp_check(int64_t V, int n_rows, int n_alt) {
    MG_REQUIRE(V >= 1 && V < (1LL << 31) && n_rows >= 0 && n_alt >= 0 && n_alt <= MG_LOGPROBS_MAX_ALT, MG_ERR_ARG,
               "logprobs: %lld entries, %d rows, %d alternatives (at most %d)", (long long)V, n_rows, n_alt,
               MG_LOGPROBS_MAX_ALT);
    return MG_OK;
}

// counters, then the parts of the most pieces of any call
extern "C" int64_t mg_logprobs_work(int64_t V, int n_rows, int n_alt) {
    TRY(lp_check(V, n_rows, n_alt));
    return LP_MAX_ROWS * 4 + LP_MAX_PARTS * (int64_t)sizeof(LpPart);
}

extern "C" int mg_logprobs(int act, const void *logits, int64_t ldl, int64_t V, int n_rows, const int32_t *ids,
                           int n_ids, int n_alt, float *lp, float *entropy, int32_t *alt_ids, float *alt_lp,
                           void *work, int64_t work_bytes, void *stream) {
    TRY(lp_check(V, n_rows, n_alt));
    MG_REQUIRE(act >= MG_ACT_F32 && act <= MG_ACT_BF16, MG_ERR_ARG, "logprobs: activation type %d", act);
    MG_REQUIRE(logits && ldl >= V && entropy && n_ids >= 0 && (n_ids == 0 || (ids && lp)) &&
                   (n_alt == 0 || (alt_ids && alt_lp)),
               MG_ERR_ARG, "logprobs: bad arguments");
    MG_REQUIRE(act_aligned(logits, act), MG_ERR_ARG, "logprobs: rows not aligned to their type");
    const int64_t need = mg_logprobs_work(V, n_rows, n_alt);
    MG_REQUIRE(work && work_bytes >= need && (reinterpret_cast<uintptr_t>(work) & 15) == 0, MG_ERR_ARG,
               "logprobs: %lld bytes of workspace (16-byte aligned), need %lld", (long long)(work ? work_bytes : 0),
               (long long)need);
    if (n_rows == 0) return MG_OK;
    LpArgs a{};
    a.x = logits;
    a.ldx = ldl;
    a.V = V;
    a.n_rows = n_rows;
    a.n_ids = n_ids;
    a.top = n_alt;
    a.ids = ids;
    a.lp = lp;
    a.entropy = entropy;
    a.top_lp = alt_lp;
    a.top_ids = alt_ids;
    a.count = static_cast<unsigned *>(work);
    a.parts = reinterpret_cast<LpPart *>(static_cast<uint8_t *>(work) + LP_MAX_ROWS * 4);
    cudaStream_t st = (cudaStream_t)stream;
    if (act == MG_ACT_F32) return logprobs_t<float>(a, st);
    if (act == MG_ACT_F16) return logprobs_t<__half>(a, st);
    return logprobs_t<__nv_bfloat16>(a, st);
}
