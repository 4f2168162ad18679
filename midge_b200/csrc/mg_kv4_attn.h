// mg_kv4_attn.h -- arguments of the attention kernels over the 4-bit cache.
#pragma once
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
    int pieces;       // pieces wanted of the whole call
    int *err;
};

// rows (query, head) that a kernel holds at a time, and the floats of one of its partial results:
// the rows' maxima and sums, then their outputs
__host__ __device__ constexpr int kv4_part_floats(int rows, int hd) { return rows * (hd + 2); }

// A sequence's share of the work.
struct Kv4Seq {
    int q0, nq, len, first, tile0, tiles;  // first: first position its first query sees
    __device__ __forceinline__ void load(const Kv4AttnArgs &a, int s) {
        q0 = a.q_start[s];
        nq = min(a.q_start[s + 1] - q0, a.max_q);
        const int l = a.kv_len[s];
        len = (int)min((int64_t)max(l, 0), a.c.cap);
        first = a.window > 0 ? max(0, len - nq - a.window + 1) : 0;
        tile0 = first >> 5;
        // at least one tile where there is a query, so that its zeros are written
        tiles = nq <= 0 ? 0 : max(1, ((len + 31) >> 5) - tile0);
    }
    __device__ __forceinline__ int groups(int gq, int rows) const { return nq <= 0 ? 0 : (nq * gq + rows - 1) / rows; }
};

}  // namespace mg
