// mg_kv4_attn.h -- arguments of the attention kernels over the 4-bit cache.
#pragma once
#include <string.h>

#include "mg_kv4.cuh"

namespace mg {

struct Kv4AttnArgs {
    Kv4 c;
    int n_heads, gq;  // gq: query heads of a key/value head
    const void *q;
    void *out;
    int64_t ldq, ldo;
    bool q_wide, out_wide;  // rows of 16-byte alignment
    const int32_t *q_start, *kv_len;
    int max_q;
    float scale;
    int window;
    const float *sinks;
    // cut units: a place for each piece's result (kv4_part_floats) and, per
    // (sequence, key/value head, row group), a counter of those that arrived
    float *parts;
    unsigned *count;
    int row_groups;   // the most row groups of a sequence
    int pieces, min_chunk;  // pieces wanted of the whole call, and the least tiles of one
    int *err;  // the workspace's status word
    // places where blocks keep the sums of what they have done of a long piece: `places` of them, as many as blocks fit
    // the GPU, each with a word that is 1 while a block has it; the few-row kernel's places lie in `rest`, the many-row
    // kernel's among the pieces' results
    unsigned *taken;
    int places;
    float *rest;
};

// A free place for this block (one thread of it).  There is one but for the time that a block takes to leave; a place
// is held to the block's end, by kv4_leave_place after a barrier of its threads.
constexpr uint32_t KV4_PLACE_POLLS = 1u << 20;
__device__ __forceinline__ int kv4_take_place(const Kv4AttnArgs &a, int err) {
    int s = blockIdx.x % a.places;
    for (uint32_t i = 0; i < KV4_PLACE_POLLS; i++, s = s + 1 < a.places ? s + 1 : 0)
        if (atomicExch(&a.taken[s], 1u) == 0u) {
            __threadfence();
            return s;
        }
    atomicExch(a.err, err);
    return s;
}
__device__ __forceinline__ void kv4_leave_place(const Kv4AttnArgs &a, int s) {
    __threadfence();
    atomicExch(&a.taken[s], 0u);
}

// rows (query, head) that a kernel holds at a time, and the floats of one of its partial results:
// the rows' maxima and sums, then their outputs
__host__ __device__ constexpr int kv4_part_floats(int rows, int hd) { return rows * (hd + 2); }

// A sequence's share of the work.
struct Kv4Seq {
    int q0, nq, len, before, first, tile0, tiles;  // before: its first query's position, first: the first it sees
    __device__ __forceinline__ void load(const Kv4AttnArgs &a, int s) {
        q0 = a.q_start[s];
        const int n = a.q_start[s + 1] - q0, l = a.kv_len[s];
        nq = min(n, a.max_q);
        len = (int)min((int64_t)max(l, 0), a.c.cap);
        before = len - n;
        first = a.window > 0 ? (int)max(0LL, (long long)before - a.window + 1) : 0;
        tile0 = first >> 5;
        // at least one tile where there is a query, so that its zeros are written
        tiles = nq <= 0 ? 0 : max(1, ((len + 31) >> 5) - tile0);
    }
    __device__ __forceinline__ int groups(int gq, int rows) const { return nq <= 0 ? 0 : (nq * gq + rows - 1) / rows; }
};

constexpr float LOG2E = 1.4426950408889634f;

// Softmax weights go to the tensor cores in f16, whose grid ends at 2^-24: a
// weight 2^(x - max) below that would vanish from the products while the sum
// still counts it, and many such make a tail that matters (32768 positions
// 17.5 nats below a first one: 8e-4 of the result).  So the reference m of a
// row's weights 2^(x - m) lies KV4_AHEAD below its largest x: weights of up to
// 2^15, nothing lost above 2^-40 of the largest.  m, sums and outputs go
// together, so the joins and sinks need no correction.  m is rounded up:
// x - m is never above KV4_AHEAD, whatever the size of x (f16 ends at 65504).
// Where m may lag behind the largest x by KV4_LAG (the many-row kernel for
// 16-bit types) it starts that much higher, and 2^-32 of the largest is kept.
constexpr float KV4_AHEAD = 15.f, KV4_LAG = 8.f;

// N consecutive elements as floats; 16 bytes at a time where the row allows
template <int N, typename T>
__device__ __forceinline__ void load_row(const T *src, bool wide, float x[N]) {
    if (wide) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < N / V; i++) {
            const uint4 v = reinterpret_cast<const uint4 *>(src)[i];
            T e[V];
            memcpy(e, &v, 16);
#pragma unroll
            for (int k = 0; k < V; k++) x[V * i + k] = to_f32(e[k]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = to_f32(src[i]);
    }
}
template <typename T> __device__ __forceinline__ void store4f(T *dst, bool wide, float4 v) {
    T e[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
    if (wide) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<uint4 *>(e);
        else *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<uint2 *>(e);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) dst[i] = e[i];
    }
}

// mg_kv4_prompt.cu: blocks of 256 rows
int64_t kv4_many_part_floats(int sms);
int kv4_attn_many(const Kv4AttnArgs &a, int hd, int act, int64_t max_kv, cudaStream_t st);

}  // namespace mg
