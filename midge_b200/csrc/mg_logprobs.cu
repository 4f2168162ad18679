// mg_logprobs.cu -- log probabilities of given tokens, the entropy of the
// distribution and its top alternatives, per logits row x of V entries:
//   z = log sum e^(x_i - m),  m = max x
//   log p_i = (x_i - m) - z,  H = z - sum e^(x_i - m) (x_i - m) / sum e^(x_i - m)
#include "mg_kv4.cuh"

namespace mg {

constexpr int LP_THREADS = 512;
constexpr int LP_MAX_TOP = 32;

struct LpArgs {
    const void *x;
    int64_t ldx, V;
    int n_rows, n_ids, top;
    const int32_t *ids;
    float *lp, *entropy, *top_lp;
    int32_t *top_ids;
};

// One block per row.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS) k_logprobs(LpArgs a) {
    __shared__ float scr[32];
    __shared__ int iscr[32];
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.ldx;
    float m = -INFINITY;
    for (int64_t i = threadIdx.x; i < a.V; i += LP_THREADS) m = fmaxf(m, to_f32(x[i]));
    m = warp_max(m);
    if (lane == 0) scr[warp] = m;
    __syncthreads();
    m = warp_max(lane < LP_THREADS / 32 ? scr[lane] : -INFINITY);
    __syncthreads();
    const float mm = m == -INFINITY ? 0.f : m;
    float s = 0.f, w = 0.f;
    for (int64_t i = threadIdx.x; i < a.V; i += LP_THREADS) {
        const float d = fmaxf(to_f32(x[i]) - mm, -1e30f), e = expf(d);
        s += e;
        w += e * d;
    }
    s = block_sum(s, scr);
    w = block_sum(w, scr);
    // no possible token: z = 0, so that every log probability is -infinity; +infinity among the logits: NaN
    const float z = m == INFINITY ? NAN : (s > 0.f ? logf(s) : 0.f);
    if (threadIdx.x == 0) a.entropy[row] = s > 0.f ? z - w / s : z;
    for (int i = threadIdx.x; i < a.n_ids; i += LP_THREADS) {
        const int32_t id = a.ids[(int64_t)row * a.n_ids + i];
        a.lp[(int64_t)row * a.n_ids + i] = id >= 0 && id < a.V ? fmaxf(to_f32(x[id]), -INFINITY) - mm - z : 0.f;
    }
    float lastv = INFINITY;
    int lasti = -1;
    for (int r = 0; r < a.top; r++) {  // the best after (lastv, lasti)
        float bv = -INFINITY;
        int bi = 0x7fffffff;
        for (int64_t i = threadIdx.x; i < a.V; i += LP_THREADS) {
            float v = to_f32(x[i]);
            if (v != v) v = -INFINITY;
            if ((v < lastv || (v == lastv && i > lasti)) && (v > bv || (v == bv && i < bi))) {
                bv = v;
                bi = (int)i;
            }
        }
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
            if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
        }
        __syncthreads();
        if (lane == 0) { scr[warp] = bv; iscr[warp] = bi; }
        __syncthreads();
        bv = scr[0];
        bi = iscr[0];
        for (int k = 1; k < LP_THREADS / 32; k++)
            if (scr[k] > bv || (scr[k] == bv && iscr[k] < bi)) { bv = scr[k]; bi = iscr[k]; }
        lastv = bv;
        lasti = bi;
        if (threadIdx.x == 0) {
            const bool any = bi != 0x7fffffff;  // fewer than `top` entries: the rest is -1, -inf
            a.top_ids[(int64_t)row * a.top + r] = any ? bi : -1;
            a.top_lp[(int64_t)row * a.top + r] = any ? bv - mm - z : -INFINITY;
        }
    }
}

}  // namespace mg

using namespace mg;

static int lp_check(int64_t V, int n_rows, int n_alt) {
    MG_REQUIRE(V >= 1 && V < (1LL << 31) && n_rows >= 0 && n_alt >= 0 && n_alt <= LP_MAX_TOP, MG_ERR_ARG,
               "logprobs: %lld entries, %d rows, %d alternatives (at most %d)", (long long)V, n_rows, n_alt, LP_MAX_TOP);
    return MG_OK;
}

extern "C" int64_t mg_logprobs_work(int64_t V, int n_rows, int n_alt) {
    TRY(lp_check(V, n_rows, n_alt));
    return 0;
}

extern "C" int mg_logprobs(int act, const void *logits, int64_t ldl, int64_t V, int n_rows, const int32_t *ids,
                           int n_ids, int n_alt, float *lp, float *entropy, int32_t *alt_ids, float *alt_lp,
                           void *work, int64_t work_bytes, void *stream) {
    TRY(lp_check(V, n_rows, n_alt));
    MG_REQUIRE(act >= MG_ACT_F32 && act <= MG_ACT_BF16, MG_ERR_ARG, "logprobs: activation type %d", act);
    MG_REQUIRE(logits && ldl >= V && entropy && n_ids >= 0 && (n_ids == 0 || (ids && lp)) &&
                   (n_alt == 0 || (alt_ids && alt_lp)),
               MG_ERR_ARG, "logprobs: bad arguments");
    const int64_t need = mg_logprobs_work(V, n_rows, n_alt);
    MG_REQUIRE(need == 0 || (work && work_bytes >= need), MG_ERR_ARG, "logprobs: %lld bytes of workspace, need %lld",
               (long long)work_bytes, (long long)need);
    if (n_rows == 0) return MG_OK;
    LpArgs a{logits, ldl, V, n_rows, n_ids, n_alt, ids, lp, entropy, alt_lp, alt_ids};
    cudaStream_t st = (cudaStream_t)stream;
    if (act == MG_ACT_F32) k_logprobs<float><<<n_rows, LP_THREADS, 0, st>>>(a);
    else if (act == MG_ACT_F16) k_logprobs<__half><<<n_rows, LP_THREADS, 0, st>>>(a);
    else k_logprobs<__nv_bfloat16><<<n_rows, LP_THREADS, 0, st>>>(a);
    MG_CHECK_LAUNCH();
    return MG_OK;
}
