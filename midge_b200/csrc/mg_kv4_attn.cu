// mg_kv4_attn.cu -- attention of new queries over the 4-bit paged cache.
//
// Query j of a sequence with n queries and kv_len cached positions (its own
// included) stands at position p = kv_len - n + j and sees the positions
// t <= p, with a window also t > p - window:
//   o = sum_t e^(s_t - m) v_t / (sum_t e^(s_t - m) [+ e^(sink - m)]),  s_t = scale q.k_t
// and 0 where it sees nothing.  The head h reads key/value head h / (n_heads / n_kv).
#include "mg_kv4.cuh"

namespace mg {

struct Kv4AttnArgs {
    Kv4 c;
    int n_heads;
    const void *q;
    void *out;
    int64_t ldq, ldo;
    const int32_t *q_start, *kv_len;
    int max_q;
    float scale;
    int window;
    const float *sinks;
};

constexpr int KA_THREADS = 128;

// Block = (key/value head, sequence, query): a tile of 128 positions at a
// time, one thread per position for the scores, one per output for the sums.
template <int HD, typename T>
__global__ void __launch_bounds__(KA_THREADS) k_kv4_attn(Kv4AttnArgs a) {
    extern __shared__ float sm[];
    const int kh = blockIdx.x, seq = blockIdx.z;
    const int gq = a.n_heads / a.c.n_kv;
    const int q0 = a.q_start[seq], nq = a.q_start[seq + 1] - q0, j = blockIdx.y;
    if (j >= nq) return;
    const int64_t len = min((int64_t)a.kv_len[seq], a.c.cap);
    const int pos = (int)len - nq + j;
    const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    float *qs = sm, *sc = qs + gq * HD, *mx = sc + gq * KA_THREADS, *den = mx + gq, *al = den + gq, *acc = al + gq;
    const T *q = static_cast<const T *>(a.q) + (int64_t)(q0 + j) * a.ldq + (int64_t)kh * gq * HD;
    for (int i = threadIdx.x; i < gq * HD; i += KA_THREADS) {
        qs[i] = to_f32(q[i]);
        acc[i] = 0.f;
    }
    for (int h = threadIdx.x; h < gq; h += KA_THREADS) {
        mx[h] = a.sinks ? a.sinks[kh * gq + h] : -INFINITY;
        den[h] = a.sinks ? 1.f : 0.f;
    }
    __syncthreads();
    for (int t0 = first & ~31; t0 <= pos; t0 += KA_THREADS) {
        const int t = t0 + threadIdx.x;
        const bool seen = t >= first && t <= pos;
        if (seen) {
            const uint8_t *tile = a.c.tile(seq, kh, t >> 5, kv4_tile_bytes(HD));
            for (int h = 0; h < gq; h++) sc[h * KA_THREADS + threadIdx.x] = 0.f;
            for (int d = 0; d < HD; d += 2) {
                const uint32_t b = tile[kv4_k_code<HD>(t & 31, d)];
                const float s = e5m2_f32(tile[kv4_k_scale<HD>(t & 31, d >> 5)]);
                const float k0 = e2m1_f32(b) * s, k1 = e2m1_f32(b >> 4) * s;
                for (int h = 0; h < gq; h++)
                    sc[h * KA_THREADS + threadIdx.x] += qs[h * HD + d] * k0 + qs[h * HD + d + 1] * k1;
            }
        }
        for (int h = 0; h < gq; h++)
            sc[h * KA_THREADS + threadIdx.x] = seen ? sc[h * KA_THREADS + threadIdx.x] * a.scale : -INFINITY;
        __syncthreads();
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int h = warp; h < gq; h += KA_THREADS / 32) {
            float m = mx[h];
            for (int i = lane; i < KA_THREADS; i += 32) m = fmaxf(m, sc[h * KA_THREADS + i]);
            m = warp_max(m);
            const float mm = m == -INFINITY ? 0.f : m;
            float s = 0.f;
            for (int i = lane; i < KA_THREADS; i += 32) {
                const float e = expf(sc[h * KA_THREADS + i] - mm);
                sc[h * KA_THREADS + i] = e;
                s += e;
            }
            s = warp_sum(s);
            if (lane == 0) {
                al[h] = expf(mx[h] - mm);
                den[h] = den[h] * al[h] + s;
                mx[h] = m;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < gq * HD; i += KA_THREADS) {
            const int h = i / HD, d = i % HD;
            float v = acc[i] * al[h];
            for (int r = 0; r < KA_THREADS; r++) {
                if (t0 + r < first || t0 + r > pos) continue;
                const uint8_t *tile = a.c.tile(seq, kh, (t0 + r) >> 5, kv4_tile_bytes(HD));
                const int p = (t0 + r) & 31;
                v += sc[h * KA_THREADS + r] * e2m1_f32(tile[kv4_v_code<HD>(p, d)] >> (d & 1) * 4) *
                     e5m2_f32(tile[kv4_v_scale<HD>(p, d >> 5)]);
            }
            acc[i] = v;
        }
        __syncthreads();
    }
    T *o = static_cast<T *>(a.out) + (int64_t)(q0 + j) * a.ldo + (int64_t)kh * gq * HD;
    for (int i = threadIdx.x; i < gq * HD; i += KA_THREADS)
        o[i] = from_f32<T>(den[i / HD] > 0.f ? acc[i] / den[i / HD] : 0.f);
}

template <typename T>
static int attn_t(const Kv4AttnArgs &a, int hd, cudaStream_t st) {
    const int gq = a.n_heads / a.c.n_kv;
    const size_t smem = ((size_t)2 * gq * hd + (size_t)gq * (KA_THREADS + 3)) * 4;
    const dim3 grid(a.c.n_kv, a.max_q, a.c.n_seqs);
    if (hd == 64) {
        TRY(ensure_smem(k_kv4_attn<64, T>, smem));
        k_kv4_attn<64, T><<<grid, KA_THREADS, smem, st>>>(a);
    } else {
        TRY(ensure_smem(k_kv4_attn<128, T>, smem));
        k_kv4_attn<128, T><<<grid, KA_THREADS, smem, st>>>(a);
    }
    MG_CHECK_LAUNCH();
    return MG_OK;
}

static int attn_check(const mg_kv4 *c, int n_heads, int max_q, int64_t max_kv, Kv4 *k) {
    TRY(kv4_take(c, k));
    MG_REQUIRE(n_heads >= 1 && n_heads % c->n_kv_heads == 0 && n_heads / c->n_kv_heads <= 64, MG_ERR_ARG,
               "kv4_attn: %d query heads over %d key/value heads (a multiple, at most 64 each)", n_heads, c->n_kv_heads);
    MG_REQUIRE(max_q >= 1 && max_q <= 65535 && max_kv >= 0 && c->n_seqs <= 65535, MG_ERR_ARG,
               "kv4_attn: max_q %d, max_kv %lld, %d sequences", max_q, (long long)max_kv, c->n_seqs);
    return MG_OK;
}

}  // namespace mg

using namespace mg;

extern "C" int64_t mg_kv4_attn_work(const mg_kv4 *c, int n_heads, int max_q, int64_t max_kv) {
    Kv4 k;
    TRY(attn_check(c, n_heads, max_q, max_kv, &k));
    return 0;
}

extern "C" int mg_kv4_attn(const mg_kv4 *c, int act, int n_heads, const void *q, int64_t ldq, const int32_t *q_start,
                           const int32_t *kv_len, int max_q, int64_t max_kv, float scale, int window,
                           const float *sinks, void *out, int64_t ldo, void *work, int64_t work_bytes, void *stream) {
    Kv4AttnArgs a{};
    TRY(attn_check(c, n_heads, max_q, max_kv, &a.c));
    const int64_t dim = (int64_t)n_heads * c->head_dim;
    MG_REQUIRE(act >= MG_ACT_F32 && act <= MG_ACT_BF16, MG_ERR_ARG, "kv4_attn: activation type %d", act);
    MG_REQUIRE(q && out && q_start && kv_len && ldq >= dim && ldo >= dim && window >= 0, MG_ERR_ARG,
               "kv4_attn: bad arguments");
    const int64_t need = mg_kv4_attn_work(c, n_heads, max_q, max_kv);
    MG_REQUIRE(need == 0 || (work && work_bytes >= need), MG_ERR_ARG, "kv4_attn: %lld bytes of workspace, need %lld",
               (long long)work_bytes, (long long)need);
    a.n_heads = n_heads;
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.max_q = max_q;
    a.scale = scale;
    a.window = window;
    a.sinks = sinks;
    cudaStream_t st = (cudaStream_t)stream;
    if (act == MG_ACT_F32) return attn_t<float>(a, c->head_dim, st);
    if (act == MG_ACT_F16) return attn_t<__half>(a, c->head_dim, st);
    return attn_t<__nv_bfloat16>(a, c->head_dim, st);
}
