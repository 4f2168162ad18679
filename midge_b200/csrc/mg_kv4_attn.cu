// mg_kv4_attn.cu -- attention of new queries over the 4-bit paged cache: the
// kernel for few query rows per key/value head (single tokens, grouped
// heads), and the entry points.
//
// Query j of a sequence with n queries and kv_len cached positions (its own
// included) stands at position p = kv_len - n + j and sees the positions
// t <= p, with a window also t > p - window:
//   o = sum_t e^(s_t - m) v_t / (sum_t e^(s_t - m) [+ e^(sink - m)]),  s_t = scale q.k_t
// and 0 where it sees nothing.  The head h reads key/value head h / gq.
#include <type_traits>

#include "mg_kv4_attn.h"
#include "mg_tc.cuh"

namespace mg {

// ------------------------------------------------------------------ few rows
// A row is a (query, head) pair of one key/value head: row r = j gq + h.  The
// kernel holds 8 rows (16 for f16 and bf16 where there are more than 8) and
// streams tiles of 32 positions:
//   * one bulk copy per tile into a ring of the warp's own (a tile with its
//     scales is contiguous in the cache), KD_NST - 1 ahead;
//   * codes -> f16 in registers (cvt.f16x2.e2m1x2, then the scale: exact),
//     straight in the order of mma.m16n8k16 fragments;
//   * both products are transposed, S^T = K Q^T and O^T = V^T P^T: the 16-row
//     operand is positions, then dimensions, and the rows are its 8 columns,
//     so no part of an MMA is empty at 8 rows (half the MMAs of Q K^T: mma.sync
//     runs at a quarter of the tcgen05 rate here, 8 cycles a scheduler);
//   * weights go from score accumulators to B fragments by movmatrix.
// f32 queries and weights go as f16 hi and lo halves in two MMAs into the
// same accumulator (22 bits; a tile's sums start from zero and are added in
// fp32, since the tensor core truncates its running sum).  f16 and bf16
// queries are scaled to f16 by a power of two per row: exact down to 2^-14 of
// the row's largest, and within 2^-25 of it below.  Their weights are rounded
// to f16, 2^-11 of a weight: an eighth of a bf16 result's own rounding, and
// as much as an f16 result's.  Weights are taken 2^15 times as large
// (KV4_AHEAD), so that small ones keep these bits too.
//
// Work: a unit is a (sequence, key/value head, row group); units of more than
// `chunk` tiles are cut into equal pieces, chunk coming from the tiles of the
// whole call, so that the pieces are alike whatever the lengths.  A block
// takes a piece, its warps the piece's tiles in turn.  A cut unit is joined by
// the last of its blocks to finish, in piece order, so results do not depend
// on the order of arrival.
//
// Measured: 8 sequences of 4096, 64 heads of 64 over 8, f32: 13.8 us (17.8 MB,
// 1.3 TB/s: launch, the pieces' table, first tiles and the join are 10 of
// them); 64 sequences of up to 32768, 32 heads of 128 over 4, bf16: 135 us
// (571 MB, 4.2 TB/s); 128 with a window of 128: 11 us (one round of blocks of
// two warps, each mostly prologue).  Bound on the long ones by latency: a
// tile of 34 HD bytes takes some 560 instructions, half of them the way from
// codes to fragments (which is why codes lie in fragment order and a warp
// shares no tile with another), in chains that the 12 to 16 warps which the
// registers allow fill to 54% of the issue slots, the tensor pipe to 25%.
constexpr int KD_NST = 4;    // ring stages of a warp
constexpr int KD_ERR = 41, KD_PLACE_ERR = 44;
constexpr int KD_WARPS_LONG = 4, KD_WARPS_SHORT = 2;  // warps of a block
// Tiles worth a piece of their own where blocks would be idle, and where they
// would not: a piece costs about as much as 16 tiles (five queries each of 16
// sequences of 1.5k to 9k: 64 tiles 61 us, 16 tiles 71; one query each of 64 of
// up to 32768: 135 either way).
constexpr int KD_MIN_CHUNK = 16, KD_LONG_CHUNK = 64;
constexpr int KD_MAX_CUT = 128;                       // pieces of a unit
// Tiles that a warp sums at a stretch in 16-bit types.  The tensor core truncates its running sum: values of one sign
// lose 1.7e-7 of theirs a tile of the warp's, 9e-5 here (measured without stretches: 6.9e-4 of 4096 tiles, 524288
// positions of each of 320 sequences).  A longer piece is done in several goes, whose sums rest in the block's place.
// The loop over goes costs 1 to 3% (16 x 5 queries 63.6 -> 65.1 us), so calls whose table holds no longer piece go
// without it.
constexpr int KD_RUN = 512;
__host__ __device__ constexpr int kd_rest_floats(int hd) { return 16 * hd / 4 * 6; }  // a place: four outputs, maximum and sum a thread
__host__ __device__ constexpr int kd_warps_sm(int hd) { return hd == 64 ? 16 : 12; }  // 128 and 168 registers a thread

enum { KD_SPLIT = 0, KD_ROWS8 = 1, KD_ROWS16 = 2 };
__host__ __device__ constexpr int kd_rows(int mode) { return mode == KD_ROWS16 ? 16 : 8; }
template <int HD> constexpr size_t kd_smem(int warps) { return (size_t)warps * KD_NST * kv4_tile_bytes(HD); }

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// the scale byte b of a word as f16x2, both halves
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
    const float2 r = fma2(f, make_float2(-1.f, -1.f), make_float2(a, b));
    lo = h2_rn(r.x, r.y);
}
// the transpose of an 8 x 8 f16 matrix held as lane (row lane / 4, columns 2 (lane % 4), + 1)
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// D = A B, nothing added
__device__ __forceinline__ void mma4_first(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma4(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    const uint32_t a[4] = {a0, a1, a2, a3};
    mma_16816(d, a, b0, b1);
}

// a / b; both below 2^32 but for caches of terabytes
__device__ __forceinline__ long long div_line(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

// keep of the four scale bytes of positions p .. p + 3 those in [first, len)
__device__ __forceinline__ uint32_t live_bytes(uint32_t w, int p, int first, int len) {
    const int hi = len - p, lo = first - p;
    if (hi < 4) w &= hi <= 0 ? 0u : (1u << (8 * hi)) - 1u;
    if (lo > 0) w &= lo >= 4 ? 0u : ~((1u << (8 * lo)) - 1u);
    return w;
}

template <int HD, int MODE, typename T, int KD_WARPS, bool GOES>
__global__ void __launch_bounds__(KD_WARPS * 32, kd_warps_sm(HD) / KD_WARPS) k_kv4_attn_few(Kv4AttnArgs a) {
    constexpr int KD_THREADS = KD_WARPS * 32;
    constexpr int ROWS = kd_rows(MODE), SETS = ROWS / 8, TB = kv4_tile_bytes(HD), KS = HD / 16, G = HD / 32;
    constexpr int MT = HD / 16;                    // O^T tiles of 16 dimensions
    constexpr int QR = MODE == KD_SPLIT ? 4 : 2;   // query registers of a k-step: b0, b1 (and their lo halves)
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[KD_WARPS][KD_NST];
    __shared__ long long s_sum[KD_WARPS];
    __shared__ int2 s_scan[KD_WARPS];
    __shared__ Kv4Seq s_q;
    __shared__ int s_seq, s_off, s_slot, s_last, s_place;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (GOES && tid == 0) s_place = -1;
    uint8_t *ring = smem + (size_t)warp * KD_NST * TB;
    if (lane == 0) {
        for (int i = 0; i < KD_NST; i++) mbar_init(&bars[warp][i], 1);
        fence_mbar_init();
    }

    // ---- the pieces: tiles of all sequences, then pieces before each sequence
    const int n = a.c.n_seqs, per = (n + KD_THREADS - 1) / KD_THREADS, s0 = tid * per, s1 = min(n, s0 + per);
    Kv4Seq q;
    long long sum = 0;
    for (int s = s0; s < s1; s++) {
        q.load(a, s);
        sum += (long long)q.tiles * q.groups(a.gq, ROWS) * a.c.n_kv;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < KD_WARPS; w++) sum += s_sum[w];
    const int chunk = (int)max((long long)a.min_chunk, div_line(sum + a.pieces - 1, a.pieces));
    auto cuts = [&](const Kv4Seq &q) { return min(KD_MAX_CUT, (q.tiles + chunk - 1) / chunk); };
    int2 mine = make_int2(0, 0);  // pieces; pieces of cut units
    for (int s = s0; s < s1; s++) {
        if (per > 1) q.load(a, s);
        const int c = cuts(q), all = c * q.groups(a.gq, ROWS) * a.c.n_kv;
        mine.x += all;
        mine.y += c > 1 ? all : 0;
    }
    int2 excl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, excl.x, o), y = __shfl_up_sync(0xffffffffu, excl.y, o);
        if (lane >= o) {
            excl.x += x;
            excl.y += y;
        }
    }
    if (lane == 31) s_scan[warp] = excl;
    __syncthreads();
    excl.x -= mine.x;
    excl.y -= mine.y;
    int total = 0;
#pragma unroll
    for (int w = 0; w < KD_WARPS; w++) {
        if (w < warp) {
            excl.x += s_scan[w].x;
            excl.y += s_scan[w].y;
        }
        total += s_scan[w].x;
    }

    uint32_t phase = 0;  // bit i: parity of ring stage i's next completion
    bool ok = true;
    [[maybe_unused]] int done = 0;  // tiles of the piece that earlier goes did
    for (int piece = blockIdx.x; piece < total;) {
        if (piece >= excl.x && piece < excl.x + mine.x) {
            int at = excl.x, slot = excl.y;
            for (int s = s0;; s++) {
                Kv4Seq qq;
                qq.load(a, s);
                const int c = cuts(qq), all = c * qq.groups(a.gq, ROWS) * a.c.n_kv;
                if (piece < at + all) {
                    s_q = qq;
                    s_seq = s;
                    s_off = piece - at;
                    s_slot = slot;
                    break;
                }
                at += all;
                slot += c > 1 ? all : 0;
            }
        }
        __syncthreads();
        const int seq = s_seq;
        const Kv4Seq q = s_q;
        const int groups = q.groups(a.gq, ROWS), ncut = cuts(q);
        const int hr = s_off / ncut, cut = s_off - hr * ncut;
        const int kh = hr / groups, rg = hr - kh * groups;
        const int ta = (int)((long long)q.tiles * cut / ncut);
        const int piece_tiles = (int)((long long)q.tiles * (cut + 1) / ncut) - ta;
        constexpr int GO = KD_WARPS * KD_RUN;  // tiles of a go
        if (GOES && tid == 0 && piece_tiles > GO && s_place < 0) s_place = kv4_take_place(a, KD_PLACE_ERR);
        const int nt = GOES ? min(GO, piece_tiles - done) : piece_tiles, tile_a = q.tile0 + ta + (GOES ? done : 0);
        const bool last_go = !GOES || nt == piece_tiles - done;
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
            if (lane == i - addr_base) {
                mbar_arrive_expect_tx(&bars[warp][i % KD_NST], TB);
                bulk_g2s(ring + (size_t)(i % KD_NST) * TB, addr, TB, &bars[warp][i % KD_NST]);
            }
        };
        look_up(0);

        // ---- the queries as B fragments (lane: row g, dimensions t HD / 4 ..); loaded before the copies wait for the table
        uint32_t qb[SETS][KS][QR];
        float own_factor[SETS];
        float x[SETS][HD / 4];
#pragma unroll
        for (int s = 0; s < SETS; s++) {
            const int r = rg * ROWS + 8 * s + g, j = r / a.gq, h = kh * a.gq + r - j * a.gq;
            if (j < q.nq) {
                load_row<HD / 4>(static_cast<const T *>(a.q) + (int64_t)(q.q0 + j) * a.ldq + (int64_t)h * HD + t * (HD / 4),
                                 a.q_wide, x[s]);
            } else {
#pragma unroll
                for (int i = 0; i < HD / 4; i++) x[s][i] = 0.f;
            }
        }
        // every piece starts at stage 0; `phase` carries the parities
#pragma unroll
        for (int i = 0; i < KD_NST - 1; i++) issue(i);
#pragma unroll
        for (int s = 0; s < SETS; s++) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 4; i++) top = fmaxf(top, fabsf(x[s][i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^-e, e = the exponent of the row's largest: the row's values are below 2 in f16
            const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
            // (with the scale's sign, so that the factor of the scores is above zero)
            const float down = __uint_as_float((254u - e) << 23) * (a.scale < 0.f ? -1.f : 1.f);
            own_factor[s] = fmaxf(fabsf(a.scale) * LOG2E * __uint_as_float(e << 23), 1e-37f);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const float x0 = x[s][4 * k] * down, x1 = x[s][4 * k + 1] * down;
                const float x2 = x[s][4 * k + 2] * down, x3 = x[s][4 * k + 3] * down;
                if constexpr (MODE == KD_SPLIT) {
                    split_h2(x0, x1, qb[s][k][0], qb[s][k][2]);
                    split_h2(x2, x3, qb[s][k][1], qb[s][k][3]);
                } else {
                    qb[s][k][0] = h2_rn(x0, x1);
                    qb[s][k][1] = h2_rn(x2, x3);
                }
            }
        }
        // ---- the rows whose scores this lane holds: 8 s + 2 t + c
        float2 m[SETS], l[SETS], factor[SETS];
        int hi[SETS][2];
#pragma unroll
        for (int s = 0; s < SETS; s++) {
            factor[s].x = __shfl_sync(0xffffffffu, own_factor[s], 8 * t);
            factor[s].y = __shfl_sync(0xffffffffu, own_factor[s], 8 * t + 4);
            m[s] = make_float2(-INFINITY, -INFINITY);
            l[s] = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int j = (rg * ROWS + 8 * s + 2 * t + c) / a.gq;
                hi[s][c] = j < q.nq ? q.before + j : -1;
            }
        }
        float o[SETS][MT][4];  // dimension 2 MT g + 2 mt (+ 1: elements 2, 3), rows 2 t, 2 t + 1
#pragma unroll
        for (int s = 0; s < SETS; s++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) o[s][i][c] = 0.f;

        // ---- a tile's work
        auto work = [&](const uint8_t *tb, int p0, auto edge) {
            constexpr bool EDGE = decltype(edge)::value;
            const uint32_t ksc = *reinterpret_cast<const uint32_t *>(tb + 32 * HD + (g * G + t * G / 4) * 4);
            // ---- scores: sc[s][u][2 j + c] = position 16 u + 2 g + j, row 8 s + 2 t + c
            float sc[SETS][2][4];
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
                const uint32_t f0 = scale_h2(ksc, 2 * u), f1 = scale_h2(ksc, 2 * u + 1);
#pragma unroll
                for (int w = 0; w < HD / 32; w++) {
                    uint32_t h0[4], h1[4];
                    e2m1x8_to_h2(kw[0][w], h0);
                    e2m1x8_to_h2(kw[1][w], h1);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        h0[k] = hmul2_u32(h0[k], f0);
                        h1[k] = hmul2_u32(h1[k], f1);
                    }
#pragma unroll
                    for (int k = 0; k < 2; k++)
#pragma unroll
                        for (int s = 0; s < SETS; s++) {
                            const uint32_t *b = qb[s][2 * w + k];
                            if (w == 0 && k == 0) mma4_first(sc[s][u], h0[0], h1[0], h0[1], h1[1], b[0], b[1]);
                            else mma4(sc[s][u], h0[2 * k], h1[2 * k], h0[2 * k + 1], h1[2 * k + 1], b[0], b[1]);
                            if constexpr (MODE == KD_SPLIT)
                                mma4(sc[s][u], h0[2 * k], h1[2 * k], h0[2 * k + 1], h1[2 * k + 1], b[2], b[3]);
                        }
                }
            }
            // ---- weights
            uint32_t pb[SETS][2][QR];
            float2 alpha[SETS];
#pragma unroll
            for (int s = 0; s < SETS; s++) {
                if (EDGE) {
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int c = 0; c < 2; c++) {
                                const int p = p0 + 16 * u + 2 * g + j;
                                const bool seen = p <= hi[s][c] && (a.window == 0 || p > hi[s][c] - a.window);
                                sc[s][u][2 * j + c] = seen ? sc[s][u][2 * j + c] : -INFINITY;
                            }
                }
                float2 top = make_float2(max3(fmaxf(sc[s][0][0], sc[s][0][2]), sc[s][1][0], sc[s][1][2]),
                                         max3(fmaxf(sc[s][0][1], sc[s][0][3]), sc[s][1][1], sc[s][1][3]));
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    top.x = fmaxf(top.x, __shfl_xor_sync(0xffffffffu, top.x, x));
                    top.y = fmaxf(top.y, __shfl_xor_sync(0xffffffffu, top.y, x));
                }
                top = fma2_up(top, factor[s], make_float2(-KV4_AHEAD, -KV4_AHEAD));
                const float2 mn = make_float2(fmaxf(m[s].x, top.x), fmaxf(m[s].y, top.y));
                float2 mm = mn;  // -infinity only where a row has seen nothing yet
                if (EDGE) mm = make_float2(mn.x == -INFINITY ? 0.f : mn.x, mn.y == -INFINITY ? 0.f : mn.y);
                alpha[s] = make_float2(ex2(m[s].x - mm.x), ex2(m[s].y - mm.y));
                m[s] = mn;
                l[s] = mul2(l[s], alpha[s]);
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float2 x = fma2(make_float2(sc[s][u][2 * j], sc[s][u][2 * j + 1]), factor[s], make_float2(-mm.x, -mm.y));
                        const float2 e = make_float2(ex2(x.x), ex2(x.y));
                        l[s] = add2(l[s], e);
                        if constexpr (MODE == KD_SPLIT) {
                            uint32_t h, r;
                            split_h2(e.x, e.y, h, r);
                            pb[s][u][j] = transpose8(h);
                            pb[s][u][2 + j] = transpose8(r);
                        } else {
                            pb[s][u][j] = transpose8(h2_rn(e.x, e.y));
                        }
                    }
            }
            if constexpr (MODE != KD_SPLIT) {
                bool same = true;
#pragma unroll
                for (int s = 0; s < SETS; s++) same = same && alpha[s].x == 1.f && alpha[s].y == 1.f;
                if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
                    for (int s = 0; s < SETS; s++)
#pragma unroll
                        for (int k = 0; k < MT; k++) {
                            const float2 x = mul2(make_float2(o[s][k][0], o[s][k][1]), alpha[s]), y = mul2(make_float2(o[s][k][2], o[s][k][3]), alpha[s]);
                            o[s][k][0] = x.x; o[s][k][1] = x.y; o[s][k][2] = y.x; o[s][k][3] = y.y;
                        }
                }
            }
            // ---- values
            [[maybe_unused]] float d[MT][4];  // f32: this tile's sums
#pragma unroll
            for (int u = 0; u < 2; u++) {
                uint32_t vs = *reinterpret_cast<const uint32_t *>(tb + 33 * HD + ((t * G + g * G / 8) * 2 + u) * 4);
                if (EDGE) vs = live_bytes(vs, p0 + 16 * u + 4 * t, q.first, q.len);
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
                    // pairs along the positions: byte b of e..: dimension 2 b, of o..: 2 b + 1; (0, 2) and (1, 3) of the quad
                    uint32_t e02[4], o02[4], e13[4], o13[4];
                    e2m1x8_to_h2((w[0][x] & 0x0F0F0F0Fu) | ((w[2][x] << 4) & 0xF0F0F0F0u), e02);
                    e2m1x8_to_h2(((w[0][x] >> 4) & 0x0F0F0F0Fu) | (w[2][x] & 0xF0F0F0F0u), o02);
                    e2m1x8_to_h2((w[1][x] & 0x0F0F0F0Fu) | ((w[3][x] << 4) & 0xF0F0F0F0u), e13);
                    e2m1x8_to_h2(((w[1][x] >> 4) & 0x0F0F0F0Fu) | (w[3][x] & 0xF0F0F0F0u), o13);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t a0 = hmul2_u32(e02[k], f02), a1 = hmul2_u32(o02[k], f02);
                        const uint32_t a2 = hmul2_u32(e13[k], f13), a3 = hmul2_u32(o13[k], f13);
                        if constexpr (MODE == KD_SPLIT) {
                            if (u == 0) mma4_first(d[4 * x + k], a0, a1, a2, a3, pb[0][u][0], pb[0][u][1]);
                            else mma4(d[4 * x + k], a0, a1, a2, a3, pb[0][u][0], pb[0][u][1]);
                            mma4(d[4 * x + k], a0, a1, a2, a3, pb[0][u][2], pb[0][u][3]);
                        } else {
#pragma unroll
                            for (int s = 0; s < SETS; s++) mma4(o[s][4 * x + k], a0, a1, a2, a3, pb[s][u][0], pb[s][u][1]);
                        }
                    }
                }
            }
            if constexpr (MODE == KD_SPLIT) {
#pragma unroll
                for (int k = 0; k < MT; k++) {
                    const float2 x = fma2(make_float2(o[0][k][0], o[0][k][1]), alpha[0], make_float2(d[k][0], d[k][1]));
                    const float2 y = fma2(make_float2(o[0][k][2], o[0][k][3]), alpha[0], make_float2(d[k][2], d[k][3]));
                    o[0][k][0] = x.x; o[0][k][1] = x.y; o[0][k][2] = y.x; o[0][k][3] = y.y;
                }
            }
        };
#pragma unroll 1
        for (int i = 0; i < wt; i++) {
            issue(i + KD_NST - 1);  // into the stage that tile i - 1 left
            const int st = i % KD_NST;
            ok = ok && mbar_wait(&bars[warp][st], (phase >> st) & 1);
            phase ^= 1u << st;
            const uint8_t *tb = ring + (size_t)st * TB;
            const int p0 = (tile_a + warp + i * KD_WARPS) * 32;
            // some row does not see some position: the last tiles, and with a window the first ones
            if (p0 + 32 > q.before + 1 || (a.window > 0 && p0 < q.before + q.nq - a.window)) work(tb, p0, std::true_type{});
            else work(tb, p0, std::false_type{});
            __syncwarp();  // the stage is read: the next issue may fill it
        }

        // ---- the warps' results joined in shared memory, each in its own drained ring: m, l, then rows of HD + 4
        constexpr int RS = HD + 4, WS = KD_NST * TB / 4;  // floats from row to row, from warp to warp
        static_assert(ROWS * (RS + 2) <= WS, "a warp's result fits its ring");
        static_assert(KD_MAX_CUT * ROWS * 2 * 4 <= KD_WARPS_SHORT * KD_NST * TB, "the factors of a joined unit fit the rings");
        float *comb = reinterpret_cast<float *>(ring);
#pragma unroll
        for (int s = 0; s < SETS; s++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int r = 8 * s + 2 * t + c;
                float sum = c ? l[s].y : l[s].x;
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                if (g == 0) {
                    comb[r] = c ? m[s].y : m[s].x;
                    comb[ROWS + r] = sum;
                }
#pragma unroll
                for (int k = 0; k < MT; k += 2)
                    *reinterpret_cast<float4 *>(comb + 2 * ROWS + r * RS + 2 * MT * g + 2 * k) =
                        make_float4(o[s][k][c], o[s][k][2 + c], o[s][k + 1][c], o[s][k + 1][2 + c]);
            }
        __syncthreads();
        const bool whole = ncut == 1;
        const float *all = reinterpret_cast<const float *>(smem);
        constexpr int PF = kv4_part_floats(ROWS, HD);
        float *parts = a.parts + (size_t)(s_slot + hr * ncut) * PF, *part = parts + (size_t)cut * PF;  // the unit's, this piece's
        for (int i = tid * 4; i < ROWS * HD; i += KD_THREADS * 4) {
            const int r = i / HD, dd = i - r * HD;
            const int row = rg * ROWS + r, j = row / a.gq, h = kh * a.gq + row - j * a.gq;
            if (j >= q.nq) continue;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < KD_WARPS; w++) M = fmaxf(M, all[w * WS + r]);
            const float mm = M == -INFINITY ? 0.f : M;
            float L = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < KD_WARPS; w++) {
                const float e = ex2(all[w * WS + r] - mm);
                const float4 v = *reinterpret_cast<const float4 *>(all + w * WS + 2 * ROWS + r * RS + dd);
                L += all[w * WS + ROWS + r] * e;
                acc.x += v.x * e; acc.y += v.y * e; acc.z += v.z * e; acc.w += v.w * e;
            }
            if (GOES && piece_tiles > GO) {  // with what rests of the goes before, or to rest
                float *at = a.rest + (size_t)s_place * kd_rest_floats(HD) + i, *ml = at - i + 16 * HD + i / 2;
                if (done > 0) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(at));
                    const float2 s = __ldcg(reinterpret_cast<const float2 *>(ml));
                    const float M2 = fmaxf(M, s.x), m2 = M2 == -INFINITY ? 0.f : M2, e = ex2(M - m2), f = ex2(s.x - m2);
                    M = M2;
                    L = L * e + s.y * f;
                    acc.x = acc.x * e + v.x * f; acc.y = acc.y * e + v.y * f; acc.z = acc.z * e + v.z * f; acc.w = acc.w * e + v.w * f;
                }
                if (!last_go) {
                    __stcg(reinterpret_cast<float4 *>(at), acc);
                    __stcg(reinterpret_cast<float2 *>(ml), make_float2(M, L));
                    continue;
                }
            }
            if (!whole) {
                *reinterpret_cast<float4 *>(part + 2 * ROWS + i) = acc;
                if (dd == 0) {
                    part[r] = M;
                    part[ROWS + r] = L;
                }
            } else {
                float f = 1.f;
                if (a.sinks) {
                    const float sk = a.sinks[h] * LOG2E, M2 = fmaxf(M, sk), m2 = M2 == -INFINITY ? 0.f : M2;
                    f = ex2(M - m2);
                    L = L * f + ex2(sk - m2);
                }
                f = L > 0.f ? f / L : 0.f;
                store4f(static_cast<T *>(a.out) + (int64_t)(q.q0 + j) * a.ldo + (int64_t)h * HD + dd, a.out_wide,
                        make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
            }
        }
        if (!whole && last_go) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                unsigned *cnt_p = a.count + ((size_t)seq * a.c.n_kv + kh) * a.row_groups + rg;
                const bool last = atomicAdd(cnt_p, 1u) + 1u == (unsigned)ncut;
                if (last) *cnt_p = 0u;  // ready for the next call
                s_last = last;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                // the pieces' maxima and sums, then their factors, in the rings
                float *mx = reinterpret_cast<float *>(smem), *ls = mx + ncut * ROWS;
                for (int i = tid; i < ncut * ROWS; i += KD_THREADS) {
                    const float *src = parts + (size_t)(i / ROWS) * PF + i % ROWS;
                    mx[i] = __ldcg(src);
                    ls[i] = __ldcg(src + ROWS);
                }
                __syncthreads();
                for (int i = tid * 4; i < ROWS * HD; i += KD_THREADS * 4) {
                    const int r = i / HD, dd = i - r * HD;
                    const int row = rg * ROWS + r, j = row / a.gq, h = kh * a.gq + row - j * a.gq;
                    if (j >= q.nq) continue;
                    const float sk = a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
                    float M = sk;
                    for (int x = 0; x < ncut; x++) M = fmaxf(M, mx[x * ROWS + r]);
                    const float mm = M == -INFINITY ? 0.f : M;
                    float L = a.sinks ? ex2(sk - mm) : 0.f;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                    for (int x = 0; x < ncut; x++) {
                        const float e = ex2(mx[x * ROWS + r] - mm);
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(parts + (size_t)x * PF + 2 * ROWS + i));
                        L += ls[x * ROWS + r] * e;
                        acc.x += v.x * e; acc.y += v.y * e; acc.z += v.z * e; acc.w += v.w * e;
                    }
                    const float f = L > 0.f ? 1.f / L : 0.f;
                    store4f(static_cast<T *>(a.out) + (int64_t)(q.q0 + j) * a.ldo + (int64_t)h * HD + dd, a.out_wide,
                            make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
                }
            }
        }
        fence_proxy_async_smem();  // the rings held the results: copies may fill them again
        __syncthreads();
        done = last_go ? 0 : done + nt;
        if (last_go) piece += gridDim.x;
    }
    if (GOES && tid == 0 && s_place >= 0) kv4_leave_place(a, s_place);
    if (!ok) {  // a wait ran out: the copies still on their way, then out
        for (int i = 0; i < KD_NST; i++) {
            mbar_wait(&bars[warp][i], ((phase >> i) & 1) ^ 1);
            mbar_wait(&bars[warp][i], (phase >> i) & 1);
        }
        if (lane == 0) atomicExch(a.err, KD_ERR);
    }
}

// How a call is cut: into one piece per block that fits the GPU, or, where
// there are so many units that the pieces would be uneven, into KD_WAVES times
// as many.  Units of a piece or less go whole, to blocks of two warps where
// there are more of them than blocks of four fit.
constexpr int KD_WAVES = 4;
struct FewCut {
    int blocks, pieces, min_chunk, warps;
};
static int few_most(int hd, int warps) { return num_sms() * (kd_warps_sm(hd) / warps); }
static FewCut few_cut(const Kv4 &c, int gq, int rows, int max_q, int64_t max_kv, int window, int hd) {
    int64_t len = max_kv < 1 ? 1 : max_kv;
    if (window > 0 && len > (int64_t)window + max_q) len = (int64_t)window + max_q;
    const int64_t units = (int64_t)c.n_seqs * c.n_kv * ceil_div((int64_t)max_q * gq, rows);
    const int64_t tiles = (len + 31) / 32 + (window > 0 ? 1 : 0), most = few_most(hd, KD_WARPS_LONG);
    FewCut f{};
    f.pieces = (int)(units * 4 <= most ? most - units : most * KD_WAVES - (units < most ? units : most));
    f.warps = tiles <= KD_MIN_CHUNK && units > most ? KD_WARPS_SHORT : KD_WARPS_LONG;
    const int64_t share = units * tiles / most;  // of a block that fits, if there were one piece for each
    f.min_chunk = (int)(share < KD_MIN_CHUNK ? KD_MIN_CHUNK : share > KD_LONG_CHUNK ? KD_LONG_CHUNK : share);
    int64_t chunk = (units * tiles + f.pieces - 1) / f.pieces;
    if (chunk < f.min_chunk) chunk = f.min_chunk;
    const int64_t blocks = units * ((tiles + chunk - 1) / chunk);
    f.blocks = (int)(blocks < (1 << 20) ? blocks : 1 << 20);
    return f;
}

template <int HD, int MODE, typename T, int WARPS, bool GOES>
static int launch_few(Kv4AttnArgs &a, const FewCut &f, cudaStream_t st) {
    a.pieces = f.pieces;
    a.min_chunk = f.min_chunk;
    a.places = few_most(HD, WARPS);
    TRY(ensure_smem(k_kv4_attn_few<HD, MODE, T, WARPS, GOES>, kd_smem<HD>(WARPS)));
    k_kv4_attn_few<HD, MODE, T, WARPS, GOES><<<f.blocks, WARPS * 32, kd_smem<HD>(WARPS), st>>>(a);
    MG_CHECK_LAUNCH();
    return MG_OK;
}
template <int HD, int MODE, typename T, int WARPS>
static int launch_few(Kv4AttnArgs &a, const FewCut &f, cudaStream_t st) {
    if constexpr (MODE != KD_SPLIT) {  // f32 adds each tile's sums in fp32
        if (a.c.cap > (int64_t)WARPS * KD_RUN * KV4_TILE) return launch_few<HD, MODE, T, WARPS, true>(a, f, st);
    }
    return launch_few<HD, MODE, T, WARPS, false>(a, f, st);
}
template <int HD, int MODE, typename T>
static int launch_few(Kv4AttnArgs &a, const FewCut &f, cudaStream_t st) {
    return f.warps == KD_WARPS_SHORT ? launch_few<HD, MODE, T, KD_WARPS_SHORT>(a, f, st)
                                     : launch_few<HD, MODE, T, KD_WARPS_LONG>(a, f, st);
}

// rows of the kernel for a call: 16 where 8 would need a second group and the type has no lo halves
static int few_mode(int act, int gq, int max_q) {
    return act == MG_ACT_F32 ? KD_SPLIT : (int64_t)gq * max_q > 8 ? KD_ROWS16 : KD_ROWS8;
}

template <typename T>
static int attn_few(Kv4AttnArgs &a, int hd, int mode, const FewCut &f, cudaStream_t st) {
    if constexpr (sizeof(T) == 4) {
        return hd == 64 ? launch_few<64, KD_SPLIT, T>(a, f, st) : launch_few<128, KD_SPLIT, T>(a, f, st);
    } else {
        if (mode == KD_ROWS8)
            return hd == 64 ? launch_few<64, KD_ROWS8, T>(a, f, st) : launch_few<128, KD_ROWS8, T>(a, f, st);
        return hd == 64 ? launch_few<64, KD_ROWS16, T>(a, f, st) : launch_few<128, KD_ROWS16, T>(a, f, st);
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

// Rows of a key/value head from which the tcgen05 kernel (two tiles of 128
// rows a block) is taken.  16 sequences of 4096, us with 48, 64 and 96 rows, f32
// at head_dim 64: few-row kernel 76, 95, 139, tcgen05 83, 85, 86; at 128: 74, 96
// against 94, 96 (48 and 64 rows); bf16: 58, 66 against 68, 70 and, at 128, 57, 67
// against 54, 54; one sequence of 8192 with 64 rows 18 to 22 against 24 to 46.
// The kernel is chosen for the whole call, by its largest number of queries.
// A call that mixes single tokens behind long caches with a prompt chunk
// sends all of them to the 256-row blocks, uncut: 63 tokens behind up to
// 32768 positions and a chunk of 512 behind 20k take 1288 us in one call, 178
// and 341 in two (f32, 64 heads of 64 over 8; bf16, 32 of 128 over 4: 717,
// 137 and 175).
constexpr int KV4_MANY_ROWS = 64;
static bool is_many(int gq, int max_q) { return (int64_t)gq * max_q > KV4_MANY_ROWS; }

// The workspace: partial results of the most pieces of any call, so that what
// is behind them lies in the same place for every call: the status word (the
// code of a wait that ran out, 0: none), the marks of taken places and the
// few-row kernel's places, and a counter per (sequence, key/value head, row
// group).  Pieces of cut units are at most twice FewCut::pieces (a unit of
// n > 1 pieces has more than n / 2 chunks); the many-row kernel has its own
// bound and no counters.
static int64_t attn_part_bytes() {
    const int64_t d64 = (int64_t)few_most(64, KD_WARPS_LONG) * kv4_part_floats(16, 64);
    const int64_t d128 = (int64_t)few_most(128, KD_WARPS_LONG) * kv4_part_floats(16, 128);
    const int64_t few = 2 * KD_WAVES * (d64 > d128 ? d64 : d128) * 4, many = kv4_many_part_floats(num_sms()) * 4;
    return few > many ? few : many;
}
constexpr int64_t KV4_STATUS_BYTES = 16;
static int attn_places() { return few_most(64, KD_WARPS_SHORT); }  // the most blocks of any kernel here at a time
static int64_t attn_rest_bytes() {
    const int64_t d64 = (int64_t)few_most(64, KD_WARPS_SHORT) * kd_rest_floats(64);
    const int64_t d128 = (int64_t)few_most(128, KD_WARPS_SHORT) * kd_rest_floats(128);
    return (d64 > d128 ? d64 : d128) * 4;
}
static int64_t attn_work(int64_t units) {
    return attn_part_bytes() + KV4_STATUS_BYTES + attn_places() * 4 + attn_rest_bytes() + units * 4;
}

}  // namespace mg

using namespace mg;

extern "C" int64_t mg_kv4_attn_work(const mg_kv4 *c, int n_heads, int max_q, int64_t max_kv) {
    Kv4 k;
    TRY(attn_check(c, n_heads, max_q, max_kv, &k));
    return attn_work((int64_t)k.n_seqs * k.n_kv * ceil_div((int64_t)max_q * (n_heads / c->n_kv_heads), 8));
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
    MG_REQUIRE(act_aligned(q, act) && act_aligned(out, act), MG_ERR_ARG, "kv4_attn: rows not aligned to their type");
    a.gq = n_heads / c->n_kv_heads;
    a.row_groups = ceil_div((int64_t)max_q * a.gq, 8);
    const int64_t need = attn_work((int64_t)a.c.n_seqs * a.c.n_kv * a.row_groups);
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
    a.err = reinterpret_cast<int *>(static_cast<uint8_t *>(work) + attn_part_bytes());
    a.taken = reinterpret_cast<unsigned *>(a.err + KV4_STATUS_BYTES / 4);
    a.rest = reinterpret_cast<float *>(a.taken + attn_places());
    a.count = reinterpret_cast<unsigned *>(reinterpret_cast<uint8_t *>(a.rest) + attn_rest_bytes());
    const int64_t size = act_size(act);
    a.q_wide = ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(ldq * size)) & 15) == 0;
    a.out_wide = ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(ldo * size)) & 15) == 0;
    cudaStream_t st = (cudaStream_t)stream;
    a.places = num_sms();  // the many-row kernel's
    if (is_many(a.gq, max_q)) return kv4_attn_many(a, c->head_dim, act, max_kv, st);
    const int mode = few_mode(act, a.gq, max_q);
    const FewCut f = few_cut(a.c, a.gq, kd_rows(mode), max_q, max_kv, window, c->head_dim);
    if (act == MG_ACT_F32) return attn_few<float>(a, c->head_dim, mode, f, st);
    if (act == MG_ACT_F16) return attn_few<__half>(a, c->head_dim, mode, f, st);
    return attn_few<__nv_bfloat16>(a, c->head_dim, mode, f, st);
}

extern "C" int mg_kv4_attn_status(void *work, int64_t work_bytes, void *stream) {
    MG_REQUIRE(work && work_bytes >= attn_work(1) && (reinterpret_cast<uintptr_t>(work) & 15) == 0, MG_ERR_ARG,
               "kv4_attn_status: %lld bytes, not a workspace of kv4_attn", (long long)(work ? work_bytes : 0));
    cudaStream_t st = (cudaStream_t)stream;
    int code = 0;
    MG_CUDA(cudaMemcpyAsync(&code, static_cast<uint8_t *>(work) + attn_part_bytes(), sizeof(int), cudaMemcpyDeviceToHost, st));
    MG_CUDA(cudaStreamSynchronize(st));
    if (!code) return MG_OK;
    MG_CUDA(cudaMemsetAsync(work, 0, (size_t)work_bytes, st));
    MG_CUDA(cudaStreamSynchronize(st));
    set_error("kv4_attn: a bounded wait timed out (code %d)", code);
    return MG_ERR_TIMEOUT;
}
