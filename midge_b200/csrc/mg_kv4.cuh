// mg_kv4.cuh -- the 4-bit paged key/value cache: its layout, its codes and
// the activation types of the operators on it.
//
// A page holds, for each key/value head, page_size / 32 tiles of 32
// positions; a tile of head_dim D (64 or 128) has G = D / 32 groups of 32
// dimensions per position and 32 D + 64 G = 34 D bytes:
//   [0, 16 D)      keys: e2m1 codes, two per byte, the even dimension low
//   [16 D, 32 D)   values, the same
//   [32 D, 33 D)   the keys' scales: an e5m2 byte per position and group
//   [33 D, 34 D)   the values' scales
// A stored number is code x scale: at most 2 + 3 significant bits, so it is
// exact in f16 (the e5m2 byte is the high byte of the scale's f16).
//
// The codes lie in the order in which a lane of an mma.m16n8k16 warp reads
// them, lane = 4 g + t.  Keys (B operand, n = position, k = dimension): the
// lane holds positions 16 u + 2 g + j and the dimensions [t D/4, (t+1) D/4).
// Values (B operand, n = dimension, k = position): the lane holds positions
// 16 u + 4 t + i, i = c + 2 s, and the dimensions [g D/8, (g+1) D/8).  A lane
// reads both in 16-byte pieces, 512 bytes per warp and piece:
//   keys   D = 64:  piece u,       16 bytes = j (2) x 8
//          D = 128: piece 2 u + j, 16 bytes
//   values D = 64:  piece u,       16 bytes = i (4) x 4
//          D = 128: piece 2 u + c, 16 bytes = s (2) x 8
// and scales in words: keys [g][group][u][j], values [t][group][u][i].
#pragma once
#include <cuda_bf16.h>

#include "mg_common.cuh"

namespace mg {

constexpr int KV4_TILE = 32;  // positions of a tile

__host__ __device__ constexpr int kv4_tile_bytes(int hd) { return 34 * hd; }

// byte of position p's (0..31) dimension d within the tile; nibble d & 1
template <int HD>
__device__ __forceinline__ int kv4_k_code(int p, int d) {
    const int u = p >> 4, g = (p >> 1) & 7, j = p & 1;
    if (HD == 64) return u * 512 + (g * 4 + (d >> 4)) * 16 + j * 8 + ((d & 15) >> 1);
    return (2 * u + j) * 512 + (g * 4 + (d >> 5)) * 16 + ((d & 31) >> 1);
}
template <int HD>
__device__ __forceinline__ int kv4_v_code(int p, int d) {
    const int u = p >> 4, t = (p >> 2) & 3, i = p & 3;
    if (HD == 64) return 16 * HD + u * 512 + ((d >> 3) * 4 + t) * 16 + i * 4 + ((d & 7) >> 1);
    return 16 * HD + (2 * u + (i & 1)) * 512 + ((d >> 4) * 4 + t) * 16 + (i >> 1) * 8 + ((d & 15) >> 1);
}
template <int HD>
__device__ __forceinline__ int kv4_k_scale(int p, int grp) {
    return 32 * HD + (((p >> 1) & 7) * (HD / 32) + grp) * 4 + ((p >> 4) << 1) + (p & 1);
}
template <int HD>
__device__ __forceinline__ int kv4_v_scale(int p, int grp) {
    return 33 * HD + ((((p >> 2) & 3) * (HD / 32) + grp) * 2 + (p >> 4)) * 4 + (p & 3);
}

__device__ __forceinline__ float e5m2_f32(uint32_t byte) { return h2f((uint16_t)(byte << 8)); }

// The scale of a group of largest magnitude `top`: the least e5m2 value s
// with 6 s >= top, from 2^-14 (the least normal; anything below half its
// least code rounds to zero, as the f16 cache flushes subnormals) to 10240
// (larger numbers saturate at 61440, where f16 would overflow); 0 for top = 0.
__device__ __forceinline__ uint32_t kv4_scale(float top) {
    if (!(top > 0.f)) return 0u;
    // an estimate of the byte from top / 6, then one step either way by exact products (6 s has 4 significant bits)
    const float est = fminf(fmaxf(top * (1.0f / 6.0f), 6.103515625e-5f), 10240.f);
    uint32_t b = (__float_as_uint(est) >> 21) - (112u << 2);
    if (b < 0x71u && e5m2_f32(b) * 6.f < top) b++;
    if (b > 4u && e5m2_f32(b - 1) * 6.f >= top) b--;
    return b;
}
// The nearest e2m1 code of x / s, ties to the even code: |x| against the
// exact products s x midpoint (s has 3 significant bits, the midpoints 3).
// A midpoint below an odd code belongs to the even one under it, so there the
// comparison is with the next number up; positive floats compare as their
// bits.  Three comparisons find the code.  s = 0 gives code 0.
struct Kv4Mids {
    int32_t m[7];
    __device__ __forceinline__ explicit Kv4Mids(float s) {
        const float k[7] = {0.25f, 0.75f, 1.25f, 1.75f, 2.5f, 3.5f, 5.f};
#pragma unroll
        for (int i = 0; i < 7; i++) m[i] = s > 0.f ? __float_as_int(k[i] * s) + (i % 2 == 0) : 0x7fffffff;
    }
};
__device__ __forceinline__ uint32_t kv4_code(float x, const Kv4Mids &t) {
    int32_t a = __float_as_int(x) & 0x7fffffff;
    a = a > 0x7f800000 ? 0 : a;  // NaN
    const bool hi = a >= t.m[3], mid = a >= (hi ? t.m[5] : t.m[1]);
    const int32_t last = hi ? (mid ? t.m[6] : t.m[4]) : (mid ? t.m[2] : t.m[0]);
    const uint32_t c = (hi ? 4u : 0u) + (mid ? 2u : 0u) + (a >= last ? 1u : 0u);
    return c | (x < 0.f ? 8u : 0u);
}

// ------------------------------------------- two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
        " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 fma2_up(float2 a, float2 b, float2 c) {  // rounded up
    float2 r;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
        " fma.rp.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// ------------------------------------------------------- activation types
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// bytes of an activation type's element, and whether a row of them can start at p (a kernel's load elsewhere would fault)
inline int act_size(int act) { return act == MG_ACT_F32 ? 4 : 2; }
inline bool act_aligned(const void *p, int act) { return reinterpret_cast<uintptr_t>(p) % act_size(act) == 0; }

// The cache as the kernels take it.  Table entries are clamped to the pool,
// so that a stale entry reads another page but never outside the pool.
struct Kv4 {
    uint8_t *pages;
    const int32_t *table;
    int64_t ld_table, head_bytes;  // head_bytes: one key/value head of one page
    int n_kv, page, n_seqs;
    int n_pages;
    int64_t cap;                   // positions the table's rows cover
    // tile of positions [32 tile, 32 tile + 32) of sequence seq, key/value head h
    __device__ __forceinline__ uint8_t *tile(int seq, int h, int tile, int tile_bytes) const {
        const int per = page >> 5, pg = tile / per;
        int id = table[(int64_t)seq * ld_table + pg];
        id = id < 0 ? 0 : (id >= n_pages ? n_pages - 1 : id);
        return pages + ((int64_t)id * n_kv + h) * head_bytes + (int64_t)(tile - pg * per) * tile_bytes;
    }
};
int kv4_take(const mg_kv4 *c, Kv4 *out);  // checks the geometry (mg_kv4.cu)

}  // namespace mg
