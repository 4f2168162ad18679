// mg_kv4.cu -- storing keys and values in the 4-bit paged cache (with the
// per-head norms and the rotation of queries and keys on the way), and
// reading stored positions back.
#include "mg_kv4.cuh"

namespace mg {

int kv4_take(const mg_kv4 *c, Kv4 *o) {
    MG_REQUIRE(c && c->pages && c->table, MG_ERR_ARG, "kv4: null cache, pages or table");
    MG_REQUIRE(c->head_dim == 64 || c->head_dim == 128, MG_ERR_ARG, "kv4: head_dim %d (64 or 128)", c->head_dim);
    MG_REQUIRE(c->n_kv_heads >= 1 && c->n_kv_heads <= 1024, MG_ERR_ARG, "kv4: %d key/value heads", c->n_kv_heads);
    MG_REQUIRE(c->page_size >= KV4_TILE && c->page_size % KV4_TILE == 0 && c->page_size <= 4096, MG_ERR_ARG,
               "kv4: page_size %d (a multiple of 32, at most 4096)", c->page_size);
    MG_REQUIRE(c->n_pages >= 1 && c->n_pages < (1LL << 31) && c->n_seqs >= 1 && c->ld_table >= 1 &&
                   c->ld_table <= (1LL << 31) / c->page_size - 1,
               MG_ERR_ARG, "kv4: %lld pages, %d sequences of %lld table entries", (long long)c->n_pages, c->n_seqs,
               (long long)c->ld_table);
    MG_REQUIRE((reinterpret_cast<uintptr_t>(c->pages) & 15) == 0, MG_ERR_ARG, "kv4: pages not 16-byte aligned");
    o->pages = static_cast<uint8_t *>(c->pages);
    o->table = c->table;
    o->ld_table = c->ld_table;
    o->head_bytes = (int64_t)(c->page_size / KV4_TILE) * kv4_tile_bytes(c->head_dim);
    o->n_kv = c->n_kv_heads;
    o->page = c->page_size;
    o->n_seqs = c->n_seqs;
    o->n_pages = (int)c->n_pages;
    o->cap = c->ld_table * c->page_size;
    return MG_OK;
}

struct AppendArgs {
    Kv4 c;
    int n_tok, n_heads;
    const void *q, *k, *v;
    int64_t ldq, ldk, ldv, ldo, rope_rows;
    const float *q_norm, *k_norm, *cos, *sin;
    float eps;
    const int32_t *seq, *pos;
    void *q_out;
};

// A thread has the dimensions [4 a, 4 a + 4) of a head and their partners
// half a head up, which the rotation pairs; HD / 8 lanes make a head and 8
// lanes a scale group.
constexpr int AP_THREADS = 256;

__device__ __forceinline__ float sticky_f32(double x) {
    // toward zero, with the last bit set when inexact: compares with every
    // number of up to 23 bits as x itself does
    const float f = __double2float_rz(x);
    return (double)f == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

template <int HD>
__device__ __forceinline__ void store4(uint8_t *tile, int p, int d, const float x[4], bool key) {
    float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!tile) return;
    const uint32_t sb = kv4_scale(top);
    const float s = e5m2_f32(sb);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) w |= kv4_code(x[i], s) << (4 * i);
    const int at = key ? kv4_k_code<HD>(p, d) : kv4_v_code<HD>(p, d);
    *reinterpret_cast<uint16_t *>(tile + at) = (uint16_t)w;
    if ((d & 31) == 0) tile[key ? kv4_k_scale<HD>(p, d >> 5) : kv4_v_scale<HD>(p, d >> 5)] = (uint8_t)sb;
}

template <int HD, typename T>
__global__ void __launch_bounds__(AP_THREADS) k_kv4_append(AppendArgs a) {
    constexpr int L = HD / 8, HALF = HD / 2;
    const int heads = a.n_heads + 2 * a.c.n_kv;
    const int64_t unit = ((int64_t)blockIdx.x * AP_THREADS + threadIdx.x) / L;
    const int d = (threadIdx.x % L) * 4;
    const int64_t tok64 = unit / heads;
    bool live = tok64 < a.n_tok;
    const int tok = live ? (int)tok64 : 0, h = live ? (int)(unit - tok64 * heads) : 0;
    const int pos = live ? a.pos[tok] : -1, seq = live ? (a.seq ? a.seq[tok] : 0) : 0;
    live = live && pos >= 0 && pos < a.c.cap && seq >= 0 && seq < a.c.n_seqs && (!a.cos || pos < a.rope_rows);
    const int kind = h < a.n_heads ? 0 : (h < a.n_heads + a.c.n_kv ? 1 : 2);
    const int hh = kind == 0 ? h : (kind == 1 ? h - a.n_heads : h - a.n_heads - a.c.n_kv);
    float x0[4], x1[4];
    {
        const T *src = static_cast<const T *>(kind == 0 ? a.q : (kind == 1 ? a.k : a.v)) +
                       (int64_t)tok * (kind == 0 ? a.ldq : (kind == 1 ? a.ldk : a.ldv)) + (int64_t)hh * HD + d;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x0[i] = live ? to_f32(src[i]) : 0.f;
            x1[i] = live ? to_f32(src[i + HALF]) : 0.f;
        }
    }
    uint8_t *tile = kind > 0 && live ? a.c.tile(seq, hh, pos >> 5, kv4_tile_bytes(HD)) : nullptr;
    const float *nw = kind == 0 ? a.q_norm : a.k_norm;
    double ss = 0.0;
    if (a.q_norm || a.k_norm) {  // the same for the whole grid
#pragma unroll
        for (int i = 0; i < 4; i++) ss += (double)x0[i] * x0[i] + (double)x1[i] * x1[i];
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    if (kind < 2) {
        // keys in 64 bits: a key that rounds to the other side of a midpoint
        // is off by a whole step of its 4 bits
        double y0[4], y1[4];
        const double inv = nw ? 1.0 / sqrt(ss / HD + (double)a.eps) : 1.0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y0[i] = nw ? x0[i] * inv * nw[d + i] : x0[i];
            y1[i] = nw ? x1[i] * inv * nw[d + HALF + i] : x1[i];
        }
        if (a.cos && live) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const double c = a.cos[(int64_t)pos * HALF + d + i], s = a.sin[(int64_t)pos * HALF + d + i];
                const double z0 = y0[i] * c - y1[i] * s, z1 = y1[i] * c + y0[i] * s;
                y0[i] = z0;
                y1[i] = z1;
            }
        }
        if (kind == 0) {
            if (live) {
                T *dst = static_cast<T *>(a.q_out) + (int64_t)tok * a.ldo + (int64_t)hh * HD + d;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    dst[i] = from_f32<T>((float)y0[i]);
                    dst[i + HALF] = from_f32<T>((float)y1[i]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x0[i] = sticky_f32(y0[i]);
                x1[i] = sticky_f32(y1[i]);
            }
        }
    }
    __syncwarp();
    store4<HD>(tile, pos & 31, d, x0, kind == 1);
    store4<HD>(tile, pos & 31, d + HALF, x1, kind == 1);
}

struct ReadArgs {
    Kv4 c;
    int n_tok;
    const int32_t *seq, *pos;
    void *k, *v;
    int64_t ldk, ldv;
};

template <int HD, typename T>
__global__ void __launch_bounds__(256) k_kv4_read(ReadArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int dim = a.c.n_kv * HD;
    const int64_t tok = i / dim;
    if (tok >= a.n_tok) return;
    const int col = (int)(i - tok * dim), h = col / HD, d = col % HD;
    const int pos = a.pos[tok], seq = a.seq ? a.seq[tok] : 0;
    float kv = 0.f, vv = 0.f;
    if (pos >= 0 && pos < a.c.cap && seq >= 0 && seq < a.c.n_seqs) {
        const uint8_t *tile = a.c.tile(seq, h, pos >> 5, kv4_tile_bytes(HD));
        const int p = pos & 31, sh = (d & 1) * 4;
        kv = e2m1_f32(tile[kv4_k_code<HD>(p, d)] >> sh) * e5m2_f32(tile[kv4_k_scale<HD>(p, d >> 5)]);
        vv = e2m1_f32(tile[kv4_v_code<HD>(p, d)] >> sh) * e5m2_f32(tile[kv4_v_scale<HD>(p, d >> 5)]);
    }
    if (a.k) static_cast<T *>(a.k)[tok * a.ldk + col] = from_f32<T>(kv);
    if (a.v) static_cast<T *>(a.v)[tok * a.ldv + col] = from_f32<T>(vv);
}

template <typename T>
static int append_t(const AppendArgs &a, int hd, cudaStream_t st) {
    const int64_t threads = (int64_t)a.n_tok * (a.n_heads + 2 * a.c.n_kv) * (hd / 8);
    const int64_t blocks = (threads + AP_THREADS - 1) / AP_THREADS;
    MG_REQUIRE(blocks < (1LL << 31), MG_ERR_ARG, "kv4_append: too many tokens x heads");
    if (hd == 64) k_kv4_append<64, T><<<(unsigned)blocks, AP_THREADS, 0, st>>>(a);
    else k_kv4_append<128, T><<<(unsigned)blocks, AP_THREADS, 0, st>>>(a);
    MG_CHECK_LAUNCH();
    return MG_OK;
}
template <typename T>
static int read_t(const ReadArgs &a, int hd, cudaStream_t st) {
    const int64_t blocks = ((int64_t)a.n_tok * a.c.n_kv * hd + 255) / 256;
    MG_REQUIRE(blocks < (1LL << 31), MG_ERR_ARG, "kv4_read: too many tokens");
    if (hd == 64) k_kv4_read<64, T><<<(unsigned)blocks, 256, 0, st>>>(a);
    else k_kv4_read<128, T><<<(unsigned)blocks, 256, 0, st>>>(a);
    MG_CHECK_LAUNCH();
    return MG_OK;
}

}  // namespace mg

using namespace mg;

extern "C" int64_t mg_kv4_page_bytes(int n_kv_heads, int head_dim, int page_size) {
    MG_REQUIRE((head_dim == 64 || head_dim == 128) && n_kv_heads >= 1 && n_kv_heads <= 1024 && page_size >= KV4_TILE &&
                   page_size % KV4_TILE == 0 && page_size <= 4096,
               MG_ERR_ARG, "kv4_page_bytes: %d heads of %d, page_size %d", n_kv_heads, head_dim, page_size);
    return (int64_t)n_kv_heads * (page_size / KV4_TILE) * kv4_tile_bytes(head_dim);
}

extern "C" int mg_kv4_append(const mg_kv4 *c, int act, int n_tok, int n_heads, const void *q, int64_t ldq,
                             const void *k, int64_t ldk, const void *v, int64_t ldv, const float *q_norm,
                             const float *k_norm, float eps, const float *rope_cos, const float *rope_sin,
                             int64_t rope_rows, const int32_t *tok_seq, const int32_t *tok_pos, void *q_out,
                             int64_t ldqo, void *stream) {
    AppendArgs a{};
    TRY(kv4_take(c, &a.c));
    const int64_t kv_dim = (int64_t)c->n_kv_heads * c->head_dim, q_dim = (int64_t)n_heads * c->head_dim;
    MG_REQUIRE(act >= MG_ACT_F32 && act <= MG_ACT_BF16, MG_ERR_ARG, "kv4_append: activation type %d", act);
    MG_REQUIRE(n_tok >= 0 && n_heads >= 0 && n_heads <= 65536 && k && v && ldk >= kv_dim && ldv >= kv_dim && tok_pos,
               MG_ERR_ARG, "kv4_append: bad arguments");
    MG_REQUIRE(n_heads == 0 || (q && q_out && ldq >= q_dim && ldqo >= q_dim), MG_ERR_ARG,
               "kv4_append: %d query heads need q and q_out rows", n_heads);
    MG_REQUIRE(!rope_cos == !rope_sin && (!rope_cos || rope_rows >= 1), MG_ERR_ARG,
               "kv4_append: rope_cos and rope_sin go together");
    MG_REQUIRE(!(eps < 0.f), MG_ERR_ARG, "kv4_append: eps %g", (double)eps);
    if (n_tok == 0) return MG_OK;
    a.n_tok = n_tok;
    a.n_heads = n_heads;
    a.q = q;
    a.k = k;
    a.v = v;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.ldo = ldqo;
    a.rope_rows = rope_rows;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.cos = rope_cos;
    a.sin = rope_sin;
    a.eps = eps;
    a.seq = tok_seq;
    a.pos = tok_pos;
    a.q_out = q_out;
    cudaStream_t st = (cudaStream_t)stream;
    if (act == MG_ACT_F32) return append_t<float>(a, c->head_dim, st);
    if (act == MG_ACT_F16) return append_t<__half>(a, c->head_dim, st);
    return append_t<__nv_bfloat16>(a, c->head_dim, st);
}

extern "C" int mg_kv4_read(const mg_kv4 *c, int act, int n_tok, const int32_t *tok_seq, const int32_t *tok_pos,
                           void *k, int64_t ldk, void *v, int64_t ldv, void *stream) {
    ReadArgs a{};
    TRY(kv4_take(c, &a.c));
    const int64_t kv_dim = (int64_t)c->n_kv_heads * c->head_dim;
    MG_REQUIRE(act >= MG_ACT_F32 && act <= MG_ACT_BF16, MG_ERR_ARG, "kv4_read: activation type %d", act);
    MG_REQUIRE(n_tok >= 0 && tok_pos && (k || v) && (!k || ldk >= kv_dim) && (!v || ldv >= kv_dim), MG_ERR_ARG,
               "kv4_read: bad arguments");
    if (n_tok == 0) return MG_OK;
    a.n_tok = n_tok;
    a.seq = tok_seq;
    a.pos = tok_pos;
    a.k = k;
    a.v = v;
    a.ldk = ldk;
    a.ldv = ldv;
    cudaStream_t st = (cudaStream_t)stream;
    if (act == MG_ACT_F32) return read_t<float>(a, c->head_dim, st);
    if (act == MG_ACT_F16) return read_t<__half>(a, c->head_dim, st);
    return read_t<__nv_bfloat16>(a, c->head_dim, st);
}
