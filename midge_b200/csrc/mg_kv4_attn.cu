// mg_kv4_attn.cu -- attention of new queries over the 4-bit paged cache: the
// kernel for few query rows per key/value head (single tokens, grouped
// heads), and the entry points.
//
// Query j of a sequence with n queries and kv_len cached positions (its own
// included) stands at position p = kv_len - n + j and sees the positions
// t <= p, with a window also t > p - window:
//   o = sum_t e^(s_t - m) v_t / (sum_t e^(s_t - m) [+ e^(sink - m)]),  s_t = scale q.k_t
// and 0 where it sees nothing.  The head h reads key/value head h / gq.
#include "mg_kernels.h"
#include "mg_kv4_attn.h"
#include "mg_tc.cuh"

namespace mg {

// ------------------------------------------------------------------ few rows
// A row is a (query, head) pair of one key/value head: row r = j gq + h.  The
// kernel holds 8 rows (f32) or 8 or 16 rows (f16, bf16) as the A operand of
// mma.m16n8k16 and streams tiles of 32 positions:
//   * one bulk copy per tile into a ring of the warp's own (a tile with its
//     scales is contiguous in the cache), NST ahead;
//   * codes -> f16 in registers (cvt.f16x2.e2m1x2, then the scale: exact),
//     straight in the order of the B fragments;
//   * scores, a running maximum and sum per row (fp32, base 2), weights as A
//     fragments from the score accumulators, no shared memory in between.
// f32 queries and weights go as f16 hi and lo halves stacked in rows g and
// g + 8 of the same MMA (22 bits; the sums of a tile start from zero and are
// added in fp32, since the tensor core truncates its running sum).  f16 and
// bf16 queries are exact in f16 after scaling by a power of two per row;
// their weights are rounded to f16 (2^-11 of a weight: a quarter of the bf16
// result's own rounding).
//
// Work: all tiles of all (sequence, key/value head, row group) in one line,
// cut evenly over the blocks, whatever the lengths; a block's warps take
// every tile of a segment in turn.  A (sequence, head) that lies in
// several blocks is joined by the last of them to finish, in block order, so
// results do not depend on the order of arrival.
constexpr int KD_NST = 4;    // ring stages of a warp
constexpr int KD_CTAS = 2;   // blocks of an SM
constexpr int KD_ERR = 41;
__host__ __device__ constexpr int kd_warps(int hd) { return hd == 64 ? 8 : 6; }  // 128 and 168 registers a thread

enum { KD_SPLIT = 0, KD_ROWS8 = 1, KD_ROWS16 = 2 };
__host__ __device__ constexpr int kd_rows(int mode) { return mode == KD_ROWS16 ? 16 : 8; }
template <int HD> constexpr size_t kd_smem() { return (size_t)kd_warps(HD) * KD_NST * kv4_tile_bytes(HD); }

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// the scale byte b of a word as f16x2 (both halves); two bytes of a word as a pair
__device__ __forceinline__ uint32_t scale_h2(uint32_t w, int b) { return __byte_perm(w, 0u, (b << 12) | (b << 4) | 0x404); }
__device__ __forceinline__ uint32_t h2_rn(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// hi = f16(x), lo = f16(x - hi), of a pair
__device__ __forceinline__ void split_h2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = h2_rn(a - f.x, b - f.y);
}

// keep of the four scale bytes of positions p .. p + 3 those in [first, len)
__device__ __forceinline__ uint32_t live_bytes(uint32_t w, int p, int first, int len) {
    const int hi = len - p, lo = first - p;
    if (hi < 4) w &= hi <= 0 ? 0u : (1u << (8 * hi)) - 1u;
    if (lo > 0) w &= lo >= 4 ? 0u : ~((1u << (8 * lo)) - 1u);
    return w;
}

template <int HD, int MODE, typename T>
__global__ void __launch_bounds__(kd_warps(HD) * 32, KD_CTAS) k_kv4_attn_few(Kv4AttnArgs a) {
    constexpr int KD_WARPS = kd_warps(HD), KD_THREADS = KD_WARPS * 32;
    constexpr int ROWS = kd_rows(MODE), TB = kv4_tile_bytes(HD), KS = HD / 16, NT = HD / 8, G = HD / 32;
    constexpr int RS = MODE == KD_ROWS16 ? 2 : 1;    // row sets of a lane: g, g + 8
    constexpr int OC = MODE == KD_ROWS16 ? 4 : 2;    // output values of a lane per n-tile
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[KD_WARPS][KD_NST];
    __shared__ long long s_scan[KD_WARPS + 1];
    __shared__ long long s_off;
    __shared__ int s_seq, s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t *ring = smem + (size_t)warp * KD_NST * TB;
    // a warp's result of a segment, in its own ring once that is drained: per row m, l, o[HD]
    float *comb = reinterpret_cast<float *>(ring);
    constexpr int COMB = KD_NST * TB / 4;  // floats from one warp's to the next
    static_assert(ROWS * (HD + 2) <= COMB, "a warp's result fits its ring");
    if (lane == 0) {
        for (int i = 0; i < KD_NST; i++) mbar_init(&bars[warp][i], 1);
        fence_mbar_init();
    }
    if (tid == 0) s_seq = -1;

    // ---- this block's share of the line of tiles
    const int n = a.c.n_seqs, per = (n + KD_THREADS - 1) / KD_THREADS;
    long long mine = 0;
    for (int s = tid * per; s < min(n, (tid + 1) * per); s++) {
        Kv4Seq q;
        q.load(a, s);
        mine += (long long)q.tiles * q.groups(a.gq, ROWS) * a.c.n_kv;
    }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < KD_WARPS; w++) {
        before += w < warp ? s_scan[w] : 0;
        total += s_scan[w];
    }
    // block b has the tiles [total b / nb, total (b + 1) / nb); tile y is block ((y + 1) nb - 1) / total's
    const long long nb = min((long long)gridDim.x, total), b = blockIdx.x;
    const long long begin = b < nb ? total * b / nb : 0, end = b < nb ? total * (b + 1) / nb : 0;
    if (begin < end) {
        const long long excl = before + incl - mine;
        if (begin >= excl && begin < excl + mine) {
            long long at = excl;
            for (int s = tid * per;; s++) {
                Kv4Seq q;
                q.load(a, s);
                const long long c = (long long)q.tiles * q.groups(a.gq, ROWS) * a.c.n_kv;
                if (begin < at + c) {
                    s_seq = s;
                    s_off = begin - at;
                    break;
                }
                at += c;
            }
        }
    }
    __syncthreads();
    if (begin >= end) return;  // the whole block; nothing is in flight

    int seq = s_seq;
    long long off = s_off, cur = begin;
    uint32_t phase = 0;  // bit i: parity of ring stage i's next completion
    bool ok = true;
    while (cur < end) {
        Kv4Seq q;
        q.load(a, seq);
        const int groups = q.groups(a.gq, ROWS);
        const long long cnt = (long long)q.tiles * groups * a.c.n_kv;
        if (off >= cnt) {
            off -= cnt;
            seq++;
            continue;
        }
        const int hr = (int)(off / q.tiles), ta = (int)(off - (long long)hr * q.tiles);
        const int kh = hr / groups, rg = hr - kh * groups;
        const int nt = (int)min((long long)(q.tiles - ta), end - cur);  // tiles of this segment
        const int tile_a = q.tile0 + ta;
        const int wt = nt > warp ? (nt - warp + KD_WARPS - 1) / KD_WARPS : 0;  // this warp's tiles of it

        // ---- bulk copies: lane i keeps the address of the warp's tile base + i
        const uint8_t *addr = nullptr;
        int addr_base = 0;
        auto look_up = [&](int base) {
            addr_base = base;
            const int i = base + lane;
            addr = i < wt ? a.c.tile(seq, kh, min(tile_a + warp + i * KD_WARPS, (int)((a.c.cap - 1) >> 5)), TB) : nullptr;
        };
        auto issue = [&](int i) {  // all lanes
            if (i >= wt || !ok) return;
            if (i - addr_base >= 32) look_up(i);
            const uint64_t p = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(addr), i - addr_base);
            if (lane == 0) {
                mbar_arrive_expect_tx(&bars[warp][i % KD_NST], TB);
                bulk_g2s(ring + (size_t)(i % KD_NST) * TB, reinterpret_cast<const void *>(p), TB, &bars[warp][i % KD_NST]);
            }
        };
        // a segment starts at stage 0 again; `phase` carries the parities
        look_up(0);
#pragma unroll
        for (int i = 0; i < KD_NST - 1; i++) issue(i);

        // ---- the rows: queries as A fragments, per-row limits and factors
        uint32_t qa[KS][MODE == KD_ROWS8 ? 2 : 4];
        float m[RS], l[RS], factor[RS];
        int hi[RS], lo[RS];
#pragma unroll
        for (int s = 0; s < RS; s++) {
            const int r = rg * ROWS + g + 8 * s, j = r / a.gq, h = kh * a.gq + r - j * a.gq;
            const bool live = j < q.nq;
            hi[s] = live ? q.len - q.nq + j : -1;
            lo[s] = a.window > 0 ? hi[s] - a.window + 1 : 0;
            m[s] = -INFINITY;
            l[s] = 0.f;
            const T *src = static_cast<const T *>(a.q) + (int64_t)(q.q0 + (live ? j : 0)) * a.ldq +
                           (int64_t)(live ? h : 0) * HD + t * (HD / 4);
            float x[HD / 4], top = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 4; i++) {
                x[i] = live ? to_f32(src[i]) : 0.f;
                top = fmaxf(top, fabsf(x[i]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^-e, e = the exponent of the row's largest: the row's values are below 2 in f16
            const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
            const float down = __uint_as_float((254u - e) << 23);
            factor[s] = a.scale * 1.4426950408889634f * __uint_as_float(e << 23);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const float x0 = x[4 * k] * down, x1 = x[4 * k + 1] * down, x2 = x[4 * k + 2] * down, x3 = x[4 * k + 3] * down;
                if constexpr (MODE == KD_SPLIT) {
                    split_h2(x0, x1, qa[k][0], qa[k][1]);
                    split_h2(x2, x3, qa[k][2], qa[k][3]);
                } else if constexpr (MODE == KD_ROWS8) {
                    qa[k][0] = h2_rn(x0, x1);
                    qa[k][1] = h2_rn(x2, x3);
                } else {
                    qa[k][s] = h2_rn(x0, x1);
                    qa[k][2 + s] = h2_rn(x2, x3);
                }
            }
        }
        float o[NT][OC];
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int c = 0; c < OC; c++) o[i][c] = 0.f;

#pragma unroll 1
        for (int i = 0; i < wt; i++) {
            issue(i + KD_NST - 1);  // into the stage that tile i - 1 left
            const int st = i % KD_NST;
            ok = ok && mbar_wait(&bars[warp][st], (phase >> st) & 1);
            phase ^= 1u << st;
            const uint8_t *tb = ring + (size_t)st * TB;
            const int p0 = (tile_a + warp + i * KD_WARPS) * 32;
            const uint32_t ksc = *reinterpret_cast<const uint32_t *>(tb + 32 * HD + (g * G + t * G / 4) * 4);
            // ---- scores of 32 positions: sc[u][j] holds columns 2t, 2t + 1 = positions 16 u + 4 t + j, + 2
            float sc[2][2][4];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                uint32_t kw[2][HD / 32];
                if constexpr (HD == 64) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(tb + u * 512 + lane * 16);
                    kw[0][0] = v.x; kw[0][1] = v.y; kw[1][0] = v.z; kw[1][1] = v.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(tb + (2 * u + j) * 512 + lane * 16);
                        kw[j][0] = v.x; kw[j][1] = v.y; kw[j][2] = v.z; kw[j][3] = v.w;
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t f = scale_h2(ksc, 2 * u + j);
                    float *d = sc[u][j];
                    d[0] = d[1] = d[2] = d[3] = 0.f;
#pragma unroll
                    for (int w = 0; w < HD / 32; w++) {
                        uint32_t h[4];
                        e2m1x8_to_h2(kw[j][w], h);
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            uint32_t af[4];
                            if constexpr (MODE == KD_ROWS8) {
                                af[0] = qa[2 * w + k][0]; af[2] = qa[2 * w + k][1]; af[1] = af[3] = 0u;
                            } else {
#pragma unroll
                                for (int c = 0; c < 4; c++) af[c] = qa[2 * w + k][c];
                            }
                            mma_16816(d, af, hmul2_u32(h[2 * k], f), hmul2_u32(h[2 * k + 1], f));
                        }
                    }
                }
            }
            // ---- weights
            // some row does not see some position: the last tiles, and with a window the first ones
            const bool edge = p0 + 32 > q.len - q.nq + 1 || (a.window > 0 && p0 < q.len - a.window);
            uint32_t pa[2][4];
            float alpha[RS];
#pragma unroll
            for (int s = 0; s < RS; s++) {
                float x[2][2][2];
                float top = -INFINITY;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            float v = (MODE == KD_SPLIT ? sc[u][j][c] + sc[u][j][2 + c] : sc[u][j][2 * s + c]) * factor[s];
                            if (edge) {
                                const int p = p0 + 16 * u + 4 * t + j + 2 * c;
                                v = p <= hi[s] && p >= lo[s] ? v : -INFINITY;
                            }
                            x[u][j][c] = v;
                            top = fmaxf(top, v);
                        }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float mn = fmaxf(m[s], top), mm = mn == -INFINITY ? 0.f : mn;
                alpha[s] = ex2(m[s] - mm);
                m[s] = mn;
                float sum = 0.f;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float e0 = ex2(x[u][j][0] - mm), e1 = ex2(x[u][j][1] - mm);
                        sum += e0 + e1;
                        if constexpr (MODE == KD_SPLIT) split_h2(e0, e1, pa[u][2 * j], pa[u][2 * j + 1]);
                        else pa[u][2 * j + s] = h2_rn(e0, e1);
                    }
                if constexpr (MODE == KD_ROWS8) pa[0][1] = pa[0][3] = pa[1][1] = pa[1][3] = 0u;
                l[s] = l[s] * alpha[s] + sum;
            }
            if constexpr (MODE != KD_SPLIT) {
                const bool same = RS == 1 ? alpha[0] == 1.f : alpha[0] == 1.f && alpha[RS - 1] == 1.f;
                if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
                    for (int k = 0; k < NT; k++)
#pragma unroll
                        for (int c = 0; c < OC; c++) o[k][c] *= alpha[c / 2];
                }
            }
            // ---- values: n-tile k is dimension (HD / 8) g + k
            float d[NT][4];
#pragma unroll
            for (int k = 0; k < NT; k++) {
                if constexpr (MODE == KD_SPLIT) d[k][0] = d[k][1] = d[k][2] = d[k][3] = 0.f;
                else if constexpr (MODE == KD_ROWS8) { d[k][0] = o[k][0]; d[k][1] = o[k][1]; d[k][2] = d[k][3] = 0.f; }
                else
#pragma unroll
                    for (int c = 0; c < 4; c++) d[k][c] = o[k][c % OC];
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                uint32_t vs = *reinterpret_cast<const uint32_t *>(tb + 33 * HD + ((t * G + g * G / 8) * 2 + u) * 4);
                if (edge) vs = live_bytes(vs, p0 + 16 * u + 4 * t, q.first, q.len);
                const uint32_t f02 = __byte_perm(vs, 0u, 0x2404), f13 = __byte_perm(vs, 0u, 0x3414);
                uint32_t w[4][HD / 64];  // words of positions 4 t + i
                if constexpr (HD == 64) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(tb + 16 * HD + u * 512 + lane * 16);
                    w[0][0] = v.x; w[1][0] = v.y; w[2][0] = v.z; w[3][0] = v.w;
                } else {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(tb + 16 * HD + (2 * u + c) * 512 + lane * 16);
                        w[c][0] = v.x; w[c][1] = v.y; w[c + 2][0] = v.z; w[c + 2][1] = v.w;
                    }
                }
#pragma unroll
                for (int x = 0; x < HD / 64; x++) {
                    // pairs along the positions: byte b of e: dimension 2 b of (0, 2); of od: dimension 2 b + 1
                    uint32_t e02[4], o02[4], e13[4], o13[4];
                    e2m1x8_to_h2((w[0][x] & 0x0F0F0F0Fu) | ((w[2][x] << 4) & 0xF0F0F0F0u), e02);
                    e2m1x8_to_h2(((w[0][x] >> 4) & 0x0F0F0F0Fu) | (w[2][x] & 0xF0F0F0F0u), o02);
                    e2m1x8_to_h2((w[1][x] & 0x0F0F0F0Fu) | ((w[3][x] << 4) & 0xF0F0F0F0u), e13);
                    e2m1x8_to_h2(((w[1][x] >> 4) & 0x0F0F0F0Fu) | (w[3][x] & 0xF0F0F0F0u), o13);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        mma_16816(d[8 * x + 2 * k], pa[u], hmul2_u32(e02[k], f02), hmul2_u32(e13[k], f13));
                        mma_16816(d[8 * x + 2 * k + 1], pa[u], hmul2_u32(o02[k], f02), hmul2_u32(o13[k], f13));
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < NT; k++) {
                if constexpr (MODE == KD_SPLIT) {
                    o[k][0] = fmaf(o[k][0], alpha[0], d[k][0] + d[k][2]);
                    o[k][1] = fmaf(o[k][1], alpha[0], d[k][1] + d[k][3]);
                } else {
#pragma unroll
                    for (int c = 0; c < OC; c++) o[k][c] = d[k][c];
                }
            }
            __syncwarp();  // the stage is read: the next issue may fill it
        }

        // ---- the warps' results joined in shared memory
#pragma unroll
        for (int s = 0; s < RS; s++) {
            l[s] += __shfl_xor_sync(0xffffffffu, l[s], 1);
            l[s] += __shfl_xor_sync(0xffffffffu, l[s], 2);
            float *dst = comb + (g + 8 * s) * (HD + 2);
            if (t == 0) {
                dst[0] = m[s];
                dst[1] = l[s];
            }
            // D columns 2 t, 2 t + 1 of n-tile k are the lanes g' = 2 t, 2 t + 1 of the B operand: dimensions (HD / 8) g' + k
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int c = 0; c < 2; c++) dst[2 + (2 * t + c) * NT + k] = o[k][2 * s + c];
        }
        __syncthreads();
        const bool whole = nt == q.tiles;
        const long long unit0 = cur - ta;  // the line's first and last tile of this (sequence, head, group)
        const float *all = reinterpret_cast<const float *>(smem);
        float *part = a.parts + ((size_t)b * 2 + (cur == begin ? 0 : 1)) * kv4_part_floats(ROWS, HD);
        for (int i = tid; i < ROWS * HD; i += KD_THREADS) {
            const int r = i / HD, dd = i - r * HD;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < KD_WARPS; w++) M = fmaxf(M, all[w * COMB + r * (HD + 2)]);
            const float mm = M == -INFINITY ? 0.f : M;
            float L = 0.f, acc = 0.f;
#pragma unroll
            for (int w = 0; w < KD_WARPS; w++) {
                const float *src = all + w * COMB + r * (HD + 2);
                const float e = ex2(src[0] - mm);
                L += src[1] * e;
                acc += src[2 + dd] * e;
            }
            const int row = rg * ROWS + r, j = row / a.gq, h = kh * a.gq + row - j * a.gq;
            if (!whole) {
                part[2 * ROWS + i] = acc;
                if (dd == 0) {
                    part[2 * r] = M;
                    part[2 * r + 1] = L;
                }
            } else if (j < q.nq) {
                if (a.sinks) {
                    const float sk = a.sinks[h] * 1.4426950408889634f, M2 = fmaxf(M, sk), m2 = M2 == -INFINITY ? 0.f : M2;
                    const float e = ex2(M - m2);
                    acc *= e;
                    L = L * e + ex2(sk - m2);
                }
                static_cast<T *>(a.out)[(int64_t)(q.q0 + j) * a.ldo + (int64_t)h * HD + dd] = from_f32<T>(L > 0.f ? acc / L : 0.f);
            }
        }
        if (!whole) {
            // the blocks that share this unit: the first one's piece is its last segment unless it begins there
            const int f = (int)(((unit0 + 1) * nb - 1) / total), e = (int)(((unit0 + q.tiles) * nb - 1) / total);
            const int f_slot = total * f / nb == unit0 ? 0 : 1;
            constexpr int PF = kv4_part_floats(ROWS, HD);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                unsigned *cnt_p = a.count + ((size_t)seq * a.c.n_kv + kh) * a.row_groups + rg;
                const bool last = atomicAdd(cnt_p, 1u) + 1u == (unsigned)(e - f + 1);
                if (last) *cnt_p = 0u;  // ready for the next call
                s_last = last;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                for (int i = tid; i < ROWS * HD; i += KD_THREADS) {
                    const int r = i / HD, dd = i - r * HD;
                    const int row = rg * ROWS + r, j = row / a.gq, h = kh * a.gq + row - j * a.gq;
                    if (j >= q.nq) continue;
                    const float sk = a.sinks ? a.sinks[h] * 1.4426950408889634f : -INFINITY;
                    const float *src = a.parts + ((size_t)f * 2 + f_slot) * PF;
                    const float *next = a.parts + (size_t)(f + 1) * 2 * PF;
                    float M = fmaxf(sk, __ldcg(src + 2 * r));
#pragma unroll 4
                    for (int x = 0; x < e - f; x++) M = fmaxf(M, __ldcg(next + (size_t)x * 2 * PF + 2 * r));
                    const float mm = M == -INFINITY ? 0.f : M;
                    float w = ex2(__ldcg(src + 2 * r) - mm);
                    float L = (a.sinks ? ex2(sk - mm) : 0.f) + __ldcg(src + 2 * r + 1) * w, acc = __ldcg(src + 2 * ROWS + i) * w;
#pragma unroll 4
                    for (int x = 0; x < e - f; x++) {
                        src = next + (size_t)x * 2 * PF;
                        w = ex2(__ldcg(src + 2 * r) - mm);
                        L += __ldcg(src + 2 * r + 1) * w;
                        acc += __ldcg(src + 2 * ROWS + i) * w;
                    }
                    static_cast<T *>(a.out)[(int64_t)(q.q0 + j) * a.ldo + (int64_t)h * HD + dd] = from_f32<T>(L > 0.f ? acc / L : 0.f);
                }
            }
        }
        fence_proxy_async_smem();  // the rings held the results: copies may fill them again
        __syncthreads();
        cur += nt;
        off += nt;
    }
    if (!ok) {  // a wait ran out: the copies still on their way, then out
        for (int i = 0; i < KD_NST; i++) {
            mbar_wait(&bars[warp][i], ((phase >> i) & 1) ^ 1);
            mbar_wait(&bars[warp][i], (phase >> i) & 1);
        }
        if (lane == 0) atomicExch(a.err, KD_ERR);
    }
}

// blocks for a call: enough to fill the GPU, and at least KD_MIN_TILES tiles each
constexpr int KD_MIN_TILES = 16;
static int few_blocks(const Kv4 &c, int gq, int rows, int max_q, int64_t max_kv, int window) {
    int64_t len = max_kv < 1 ? 1 : max_kv;
    if (window > 0 && len > (int64_t)window + max_q) len = (int64_t)window + max_q;
    const int64_t units = (int64_t)c.n_seqs * c.n_kv * ceil_div((int64_t)max_q * gq, rows);
    const int64_t tiles = units * ((len + 31) / 32 + (window > 0 ? 1 : 0));
    const int64_t most = (int64_t)num_sms() * KD_CTAS;
    const int64_t want = (tiles + KD_MIN_TILES - 1) / KD_MIN_TILES;
    return (int)(want < most ? want : most);
}

template <int HD, int MODE, typename T>
static int launch_few(Kv4AttnArgs &a, int blocks, cudaStream_t st) {
    TRY(ensure_smem(k_kv4_attn_few<HD, MODE, T>, kd_smem<HD>()));
    k_kv4_attn_few<HD, MODE, T><<<blocks, kd_warps(HD) * 32, kd_smem<HD>(), st>>>(a);
    MG_CHECK_LAUNCH();
    return MG_OK;
}

// rows of the kernel for a call: 16 where 8 would need a second group and the type has no lo halves
static int few_mode(int act, int gq, int max_q) {
    return act == MG_ACT_F32 ? KD_SPLIT : (int64_t)gq * max_q > 8 ? KD_ROWS16 : KD_ROWS8;
}

template <typename T>
static int attn_few(Kv4AttnArgs &a, int hd, int mode, int blocks, cudaStream_t st) {
    if constexpr (sizeof(T) == 4) {
        return hd == 64 ? launch_few<64, KD_SPLIT, T>(a, blocks, st) : launch_few<128, KD_SPLIT, T>(a, blocks, st);
    } else {
        if (mode == KD_ROWS8)
            return hd == 64 ? launch_few<64, KD_ROWS8, T>(a, blocks, st) : launch_few<128, KD_ROWS8, T>(a, blocks, st);
        return hd == 64 ? launch_few<64, KD_ROWS16, T>(a, blocks, st) : launch_few<128, KD_ROWS16, T>(a, blocks, st);
    }
}

static int attn_check(const mg_kv4 *c, int n_heads, int max_q, int64_t max_kv, Kv4 *k) {
    TRY(kv4_take(c, k));
    MG_REQUIRE(n_heads >= 1 && n_heads % c->n_kv_heads == 0 && n_heads / c->n_kv_heads <= 64, MG_ERR_ARG,
               "kv4_attn: %d query heads over %d key/value heads (a multiple, at most 64 each)", n_heads, c->n_kv_heads);
    MG_REQUIRE(max_q >= 1 && max_q <= 65535 && max_kv >= 0 && c->n_seqs <= 65535, MG_ERR_ARG,
               "kv4_attn: max_q %d, max_kv %lld, %d sequences", max_q, (long long)max_kv, c->n_seqs);
    return MG_OK;
}

// The workspace: partial results for the most blocks of any call, so that
// the counters behind them lie in the same place for every call, and a
// counter per (sequence, key/value head, row group).
constexpr int64_t attn_part_bytes(int sms) { return (int64_t)sms * KD_CTAS * 2 * kv4_part_floats(16, 128) * 4; }
static int64_t attn_work(const Kv4 &c, int groups) {
    return attn_part_bytes(num_sms()) + (int64_t)c.n_seqs * c.n_kv * groups * 4;
}

}  // namespace mg

using namespace mg;

extern "C" int64_t mg_kv4_attn_work(const mg_kv4 *c, int n_heads, int max_q, int64_t max_kv) {
    Kv4 k;
    TRY(attn_check(c, n_heads, max_q, max_kv, &k));
    return attn_work(k, ceil_div((int64_t)max_q * (n_heads / c->n_kv_heads), 8));
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
    a.gq = n_heads / c->n_kv_heads;
    a.row_groups = ceil_div((int64_t)max_q * a.gq, 8);
    const int64_t need = attn_work(a.c, a.row_groups);
    MG_REQUIRE(work && work_bytes >= need && (reinterpret_cast<uintptr_t>(work) & 15) == 0, MG_ERR_ARG,
               "kv4_attn: %lld bytes of workspace (16-byte aligned), need %lld", (long long)(work ? work_bytes : 0), (long long)need);
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
    a.parts = static_cast<float *>(work);
    a.count = reinterpret_cast<unsigned *>(static_cast<uint8_t *>(work) + attn_part_bytes(num_sms()));
    a.err = stream_error_word();
    MG_REQUIRE(a.err, MG_ERR_OOM, "kv4_attn: no error word");
    cudaStream_t st = (cudaStream_t)stream;
    const int mode = few_mode(act, a.gq, max_q);
    const int blocks = few_blocks(a.c, a.gq, kd_rows(mode), max_q, max_kv, window);
    if (act == MG_ACT_F32) return attn_few<float>(a, c->head_dim, mode, blocks, st);
    if (act == MG_ACT_F16) return attn_few<__half>(a, c->head_dim, mode, blocks, st);
    return attn_few<__nv_bfloat16>(a, c->head_dim, mode, blocks, st);
}
