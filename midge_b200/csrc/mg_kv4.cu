// mg_kv4.cu -- storing keys and values in the 4-bit paged cache (with the
// per-head norms and the rotation of queries and keys on the way), and
// reading stored positions back.
#include <string.h>

#include <initializer_list>
#include <type_traits>

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
    int64_t ldq, ldk, ldv, ldo;
    int rope_rows;
    const float *q_norm, *k_norm, *cos, *sin;
    float eps;
    const int32_t *seq, *pos;
    void *q_out;
    int cache_shares;  // blocks of a token that have keys and values
    bool wide;         // every row, the rotation and the norm weights of 16-byte alignment
};

// Block = a token and a share of its heads.  A thread has V = 16 bytes of
// dimensions [V a, V a + V) of a head and their partners half a head up, which
// the rotation pairs: HD / 2V lanes make a head, 32 / V lanes a scale group.
// Blocks of queries and blocks of keys and values differ (the latter first:
// they take longer), so that no block has both.
// Bound: HBM (rows in, queries out; the codes are a tenth), which takes many
// threads in flight.  Measured with the read back: 4096 tokens, 64 + 2 x 8 heads
// of 64, f32: 37 us (165 MB, 4.5 TB/s; the read 4.4); 8191 tokens, 32 + 2 x 4
// heads of 128 with norms, bf16: 51 us (181 MB, 3.5 TB/s: the norms and the
// keys' 64-bit arithmetic share the issue slots; the read 6.1); 8 tokens: 5.3
// us, two launches of two dependent loads.  A query head a thread: 39 and 59 us, three or four heads 36
// and 63 or more (16-bit rows spill).
constexpr int AP_THREADS = 128, AP_HEADS = 2;

__device__ __forceinline__ float sticky_f32(double x) {
    // toward zero, with the last bit set when inexact: compares with every
    // number of up to 23 bits as x itself does
    const float f = __double2float_rz(x);
    return (double)f == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// 16 bytes of a row as numbers, and back
template <typename T>
__device__ __forceinline__ void numbers(const uint4 &q, float *x) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (std::is_same<T, float>::value) {
            x[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        } else {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 packed(const float *x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (std::is_same<T, float>::value) {
            w[i] = __float_as_uint(x[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int V, bool WIDE, typename T>
__device__ __forceinline__ void load_v(const T *src, float x[V]) {
    if constexpr (WIDE) {
        numbers<T>(__ldg(reinterpret_cast<const uint4 *>(src)), x);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = to_f32(src[i]);
    }
}
template <int V, bool WIDE>
__device__ __forceinline__ void load_f32(const float *src, float x[V]) {
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 v = __ldg(reinterpret_cast<const float4 *>(src + i));
            x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = src[i];
    }
}
template <int V, bool WIDE, typename T>
__device__ __forceinline__ void store_v(T *dst, const float x[V]) {
    if constexpr (WIDE) {
        *reinterpret_cast<uint4 *>(dst) = packed<T>(x);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) dst[i] = from_f32<T>(x[i]);
    }
}

// V numbers of dimensions d .. of position p (0..31 of the tile) stored by the
// lanes of `mask`, whole scale groups of one head
template <int HD, int V>
__device__ __forceinline__ void store_codes(uint8_t *tile, int p, int d, const float x[V], bool key, unsigned mask) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
    for (int o = 16 / V; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, o));
    const uint32_t sb = kv4_scale(top);
    const Kv4Mids m(e5m2_f32(sb));
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < V; i++) w |= kv4_code(x[i], m) << (4 * i);
    const int at = key ? kv4_k_code<HD>(p, d) : kv4_v_code<HD>(p, d);
    if constexpr (V == 8) {
        *reinterpret_cast<uint32_t *>(tile + at) = w;
    } else {  // two lanes' codes together
        w |= __shfl_xor_sync(mask, w, 1) << 16;
        if ((d & 7) == 0) *reinterpret_cast<uint32_t *>(tile + at) = w;
    }
    if ((d & 31) == 0) tile[key ? kv4_k_scale<HD>(p, d >> 5) : kv4_v_scale<HD>(p, d >> 5)] = (uint8_t)sb;
}

// Queries of a token: a thread has its dimensions of AP_HEADS heads, with one
// load of the rotation and the weights for all.
template <int HD, typename T, bool WIDE>
__device__ __forceinline__ void append_queries(const AppendArgs &a, int share) {
    constexpr int V = 16 / sizeof(T), HALF = HD / 2, L = HALF / V;
    const int tok = blockIdx.x, d = (threadIdx.x % L) * V, step = blockDim.x / L;
    const int h0 = share * step * AP_HEADS + threadIdx.x / L;
    const int pos = a.pos[tok], seq = a.seq ? a.seq[tok] : 0;
    const T *src = static_cast<const T *>(a.q) + (int64_t)tok * a.ldq + d;
    float x0[AP_HEADS][V], x1[AP_HEADS][V];
#pragma unroll
    for (int k = 0; k < AP_HEADS; k++) {
        const int h = min(h0 + k * step, a.n_heads - 1);
        load_v<V, WIDE>(src + (int64_t)h * HD, x0[k]);
        load_v<V, WIDE>(src + (int64_t)h * HD + HALF, x1[k]);
    }
    if (pos < 0 || pos >= a.c.cap || seq < 0 || seq >= a.c.n_seqs || (a.cos && pos >= a.rope_rows)) return;
    if (a.q_norm) {
        float w0[V], w1[V];
        load_f32<V, WIDE>(a.q_norm + d, w0);
        load_f32<V, WIDE>(a.q_norm + d + HALF, w1);
#pragma unroll
        for (int k = 0; k < AP_HEADS; k++) {
            auto mean_square = [&] {
                float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float2 v = make_float2(x0[k][i], x1[k][i]);
                    s2 = fma2(v, v, s2);
                }
                float ss = s2.x + s2.y;
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
                return ss * (1.0f / HD);
            };
            float mean = mean_square() + a.eps;
            // squares beyond fp32 (or, with an eps of nothing, below it): the head times a power of two, which drops out again
            const bool far = !(mean < 0x1p127f) || mean < 0x1p-100f;
            if (__any_sync(~0u, far)) {
                const float f = !far ? 1.f : mean < 1.f ? 0x1p100f : 0x1p-80f;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    x0[k][i] *= f;
                    x1[k][i] *= f;
                }
                mean = mean_square() + a.eps * f * f;
            }
            float inv = rsqrtf(mean);  // and a Newton step
            inv = mean > 0.f && mean < INFINITY ? inv * fmaf(-0.5f * mean * inv, inv, 1.5f) : inv;
            const float2 i2 = make_float2(inv, inv);
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 y0 = mul2(mul2(make_float2(x0[k][i], x0[k][i + 1]), i2), make_float2(w0[i], w0[i + 1]));
                const float2 y1 = mul2(mul2(make_float2(x1[k][i], x1[k][i + 1]), i2), make_float2(w1[i], w1[i + 1]));
                x0[k][i] = y0.x; x0[k][i + 1] = y0.y;
                x1[k][i] = y1.x; x1[k][i + 1] = y1.y;
            }
        }
    }
    if (a.cos) {
        float co[V], si[V];
        load_f32<V, WIDE>(a.cos + (int64_t)pos * HALF + d, co);
        load_f32<V, WIDE>(a.sin + (int64_t)pos * HALF + d, si);
#pragma unroll
        for (int k = 0; k < AP_HEADS; k++)
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 a0 = make_float2(x0[k][i], x0[k][i + 1]), a1 = make_float2(x1[k][i], x1[k][i + 1]);
                const float2 c = make_float2(co[i], co[i + 1]), s = make_float2(si[i], si[i + 1]);
                const float2 z0 = fma2(a0, c, mul2(a1, make_float2(-s.x, -s.y))), z1 = fma2(a1, c, mul2(a0, s));
                x0[k][i] = z0.x; x0[k][i + 1] = z0.y;
                x1[k][i] = z1.x; x1[k][i + 1] = z1.y;
            }
    }
    T *dst = static_cast<T *>(a.q_out) + (int64_t)tok * a.ldo + d;
#pragma unroll
    for (int k = 0; k < AP_HEADS; k++) {
        const int h = h0 + k * step;
        if (h < a.n_heads) {
            store_v<V, WIDE>(dst + (int64_t)h * HD, x0[k]);
            store_v<V, WIDE>(dst + (int64_t)h * HD + HALF, x1[k]);
        }
    }
}

// Keys and values of a token: whole scale groups of a head, the lanes of `mask`.
template <int HD, typename T, bool WIDE>
__device__ __forceinline__ void append_cache(const AppendArgs &a, int share) {
    constexpr int V = 16 / sizeof(T), HALF = HD / 2, L = HALF / V;
    const int tok = blockIdx.x, d = (threadIdx.x % L) * V;
    const int h = share * (blockDim.x / L) + threadIdx.x / L;
    const unsigned mask = L == 32 ? ~0u : ((1u << L) - 1u) << ((threadIdx.x & 31) / L * L);
    if (h >= 2 * a.c.n_kv) return;
    const int pos = a.pos[tok], seq = a.seq ? a.seq[tok] : 0;
    const bool key = h < a.c.n_kv;
    const int hh = key ? h : h - a.c.n_kv;
    const T *src = static_cast<const T *>(key ? a.k : a.v) + (int64_t)tok * (key ? a.ldk : a.ldv) + (int64_t)hh * HD + d;
    float x0[V], x1[V];
    load_v<V, WIDE>(src, x0);
    load_v<V, WIDE>(src + HALF, x1);
    if (pos < 0 || pos >= a.c.cap || seq < 0 || seq >= a.c.n_seqs || (a.cos && pos >= a.rope_rows)) return;
    uint8_t *tile = a.c.tile(seq, hh, pos >> 5, kv4_tile_bytes(HD));
    if (key && (a.k_norm || a.cos)) {
        // keys in 64 bits: a key that rounds to the other side of a midpoint is off by a whole step of its 4 bits
        double inv = 1.0;
        if (a.k_norm) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < V; i++) ss += (double)x0[i] * x0[i] + (double)x1[i] * x1[i];
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
            inv = 1.0 / sqrt(ss / HD + (double)a.eps);
        }
#pragma unroll
        for (int j = 0; j < V; j += 4) {  // four at a time: 64-bit values of all would not fit the registers
            float co[4], si[4], w0[4], w1[4];
            if (a.cos) {
                load_f32<4, WIDE>(a.cos + (int64_t)pos * HALF + d + j, co);
                load_f32<4, WIDE>(a.sin + (int64_t)pos * HALF + d + j, si);
            }
            if (a.k_norm) {
                load_f32<4, WIDE>(a.k_norm + d + j, w0);
                load_f32<4, WIDE>(a.k_norm + d + HALF + j, w1);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                double y0 = x0[j + i], y1 = x1[j + i];
                if (a.k_norm) {
                    y0 = y0 * inv * w0[i];
                    y1 = y1 * inv * w1[i];
                }
                if (a.cos) {
                    const double c = co[i], s = si[i], z = y0 * c - y1 * s;
                    y1 = y1 * c + y0 * s;
                    y0 = z;
                }
                x0[j + i] = sticky_f32(y0);
                x1[j + i] = sticky_f32(y1);
            }
            if (V > 4) __syncwarp(mask);
        }
    }
    store_codes<HD, V>(tile, pos & 31, d, x0, key, mask);
    store_codes<HD, V>(tile, pos & 31, d + HALF, x1, key, mask);
}

template <int HD, typename T, bool WIDE>
__global__ void __launch_bounds__(AP_THREADS, 8) k_kv4_append(AppendArgs a) {
    if ((int)blockIdx.y < a.cache_shares) append_cache<HD, T, WIDE>(a, blockIdx.y);
    else append_queries<HD, T, WIDE>(a, blockIdx.y - a.cache_shares);
}

struct ReadArgs {
    Kv4 c;
    int n_tok;
    const int32_t *seq, *pos;
    void *k, *v;
    int64_t ldk, ldv;
    bool wide;
};

// thread = eight dimensions of a token's key and value head.  Bound: HBM and
// latency (8191 tokens of 4 heads of 128 to bf16: 6.1 us, 21 MB; 8 tokens 2.5
// us, a launch)
template <int HD, typename T, bool WIDE>
__global__ void __launch_bounds__(256) k_kv4_read(ReadArgs a) {
    constexpr int L = HD / 8;
    const int per = a.c.n_kv * L;
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    const uint32_t tok = i / per;
    if (tok >= (uint32_t)a.n_tok) return;
    const int r = (int)(i - tok * per), h = r / L, d = (r - h * L) * 8;
    const int pos = a.pos[tok], seq = a.seq ? a.seq[tok] : 0;
    const bool in = pos >= 0 && pos < a.c.cap && seq >= 0 && seq < a.c.n_seqs;
    const uint8_t *tile = in ? a.c.tile(seq, h, pos >> 5, kv4_tile_bytes(HD)) : nullptr;
    const int p = pos & 31;
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
        T *dst = static_cast<T *>(kv ? a.v : a.k);
        if (!dst) continue;
        dst += (int64_t)tok * (kv ? a.ldv : a.ldk) + h * HD + d;
        uint32_t c[4] = {0u, 0u, 0u, 0u};
        float s = 0.f;
        if (in) {
            e2m1x8_to_h2(*reinterpret_cast<const uint32_t *>(tile + (kv ? kv4_v_code<HD>(p, d) : kv4_k_code<HD>(p, d))), c);
            s = e5m2_f32(tile[kv ? kv4_v_scale<HD>(p, d >> 5) : kv4_k_scale<HD>(p, d >> 5)]);
        }
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&c[j]));
            x[2 * j] = f.x * s;
            x[2 * j + 1] = f.y * s;
        }
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < 8; j += V) store_v<V, WIDE>(dst + j, x + j);
    }
}

template <typename T>
static int append_t(AppendArgs &a, int hd, cudaStream_t st) {
    // blocks of up to AP_THREADS threads, smaller ones where that leaves the GPU empty
    const int lanes = hd / 2 / (16 / (int)sizeof(T)), heads = a.n_heads + 2 * a.c.n_kv;
    int threads = AP_THREADS;
    while (threads > 64 && (int64_t)a.n_tok * ceil_div((int64_t)heads * lanes, threads) < num_sms()) threads /= 2;
    a.cache_shares = ceil_div((int64_t)2 * a.c.n_kv * lanes, threads);
    const dim3 grid(a.n_tok, (unsigned)(a.cache_shares + ceil_div((int64_t)ceil_div(a.n_heads, AP_HEADS) * lanes, threads)));
    if (hd == 64) {
        if (a.wide) k_kv4_append<64, T, true><<<grid, threads, 0, st>>>(a);
        else k_kv4_append<64, T, false><<<grid, threads, 0, st>>>(a);
    } else {
        if (a.wide) k_kv4_append<128, T, true><<<grid, threads, 0, st>>>(a);
        else k_kv4_append<128, T, false><<<grid, threads, 0, st>>>(a);
    }
    MG_CHECK_LAUNCH();
    return MG_OK;
}
template <typename T>
static int read_t(const ReadArgs &a, int hd, cudaStream_t st) {
    const int64_t threads = (int64_t)a.n_tok * a.c.n_kv * (hd / 8);
    MG_REQUIRE(threads < (1LL << 32) - 256, MG_ERR_ARG, "kv4_read: too many tokens");
    const unsigned blocks = (unsigned)((threads + 255) / 256);
    if (hd == 64) {
        if (a.wide) k_kv4_read<64, T, true><<<blocks, 256, 0, st>>>(a);
        else k_kv4_read<64, T, false><<<blocks, 256, 0, st>>>(a);
    } else {
        if (a.wide) k_kv4_read<128, T, true><<<blocks, 256, 0, st>>>(a);
        else k_kv4_read<128, T, false><<<blocks, 256, 0, st>>>(a);
    }
    MG_CHECK_LAUNCH();
    return MG_OK;
}

// every pointer and row stride (in elements of `size` bytes) of 16-byte alignment
static bool wide_rows(int size, std::initializer_list<const void *> p, std::initializer_list<int64_t> ld) {
    for (const void *x : p)
        if (reinterpret_cast<uintptr_t>(x) & 15) return false;
    for (int64_t l : ld)
        if ((l * size) & 15) return false;
    return true;
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
    MG_REQUIRE(act_aligned(q, act) && act_aligned(k, act) && act_aligned(v, act) && act_aligned(q_out, act), MG_ERR_ARG,
               "kv4_append: rows not aligned to their type");
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
    a.rope_rows = (int)(rope_rows < 0x7fffffff ? rope_rows : 0x7fffffff);
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.cos = rope_cos;
    a.sin = rope_sin;
    a.eps = eps;
    a.seq = tok_seq;
    a.pos = tok_pos;
    a.q_out = q_out;
    const int size = act_size(act);
    a.wide = wide_rows(size, {k, v}, {ldk, ldv}) && (n_heads == 0 || wide_rows(size, {q, q_out}, {ldq, ldqo})) &&
             wide_rows(4, {q_norm, k_norm, rope_cos, rope_sin}, {});
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
    MG_REQUIRE(act_aligned(k, act) && act_aligned(v, act), MG_ERR_ARG, "kv4_read: rows not aligned to their type");
    if (n_tok == 0) return MG_OK;
    a.n_tok = n_tok;
    a.seq = tok_seq;
    a.pos = tok_pos;
    a.k = k;
    a.v = v;
    a.ldk = ldk;
    a.ldv = ldv;
    const int size = act_size(act);
    a.wide = (!k || wide_rows(size, {k}, {ldk})) && (!v || wide_rows(size, {v}, {ldv}));
    cudaStream_t st = (cudaStream_t)stream;
    if (act == MG_ACT_F32) return read_t<float>(a, c->head_dim, st);
    if (act == MG_ACT_F16) return read_t<__half>(a, c->head_dim, st);
    return read_t<__nv_bfloat16>(a, c->head_dim, st);
}
