// mg_kv4_prompt.cu -- attention of many new queries over the 4-bit paged
// cache (prompt chunks, several drafted tokens) on the 5th-generation tensor
// cores.
//
// A block has 256 rows ((query, head) pairs of one key/value head, two tiles
// of 128) and walks the cache in blocks of KVB positions:
//   warps 0-3, 4-7    softmax of tile 0 / 1, thread = row: S from TMEM, row
//                     maximum, weights as f16 back into TMEM over S
//   warps 8-14        codes -> f16 K and V tiles in 128-byte-swizzled shared
//                     memory (cvt.f16x2.e2m1x2 and the scale: exact), once
//                     for both tiles
//   warp 15           issues the MMAs: S = Q K^T (both from shared memory),
//                     O += P V (P from TMEM)
// The two tiles alternate: while one tile's MMAs run the other's softmax has
// the MUFU (16 ex2 per cycle and SM, so 2048 cycles for 256 x 128 weights;
// the MMAs of the same take some 500 for S and 700 for P V at head_dim 64, twice
// that in f32).
// f32: queries and weights go as f16 hi + lo, two MMAs each (22 bits), and O
// stays in registers: each block's product starts from zero and is added in
// fp32, since the tensor core truncates its running sum.  f16 and bf16: a
// query is exact in f16 after scaling by a power of two per row (what falls
// below f16's range is 2^-24 of the row's largest), weights are rounded to
// f16 (2^-11, an eighth of the result's own rounding in bf16 and like it in f16)
// and O accumulates in TMEM for KP_RUN blocks at a time: truncated sums, off by
// 9e-5 at worst.
//
// Measured, one sequence of 4096 new tokens, 64 heads of 64 over 8, f32:
// 0.33 ms = 414 TFLOP/s, 830 of f16 MMAs; 3 x 1009 tokens behind 5k to 16k,
// 32 heads of 128 over 4, bf16: 0.49 ms = 1.03 PFLOP/s.  A block of 128 positions
// takes some 4000 cycles: bound by the chain S -> maximum -> weights -> P V of
// a tile, of which the other tile hides about half, then by the MUFU; P V of a
// block's first half starts while the weights of the second are worked out
// (340 and 507 us without; quarters measured the same as halves); a block of
// rows adds some 10 us of its own at start and end.  Blocks of 64 positions
// measured 6% slower on the first and 24% on the second.
#include <type_traits>

#include "mg_kv4_attn.h"
#include "mg_tc.cuh"

namespace mg {

constexpr int KP_ROWS = 256;        // rows of a block
constexpr int KP_THREADS = 512;
constexpr int KP_DEQ = 7;           // warps 8-14
constexpr int KP_ERR = 42, KP_PLACE_ERR = 43;
// Blocks that 16-bit types sum in TMEM at a stretch, a power of two: 9e-5 lost at worst, a fifth of f16's rounding.  Three
// chunks behind 5k to 16k: 536 us as with sums of any length, with half as many 545.
constexpr int KP_RUN = 128;

template <int HD, bool SPLIT>
struct KpCfg {
    static constexpr int KVB = HD == 128 && SPLIT ? 64 : 128;  // positions of a block
    static constexpr int PLANES = HD / 64;                     // 64 dimensions = 128 bytes a row
    static constexpr int Q_HALF = PLANES * 128 * 128;          // bytes of one tile's hi (or lo) queries
    static constexpr int Q_TILE = Q_HALF * (SPLIT ? 2 : 1);
    static constexpr int KV_STAGE = PLANES * KVB * 128;        // bytes of a K (or V) stage
    static constexpr int SMEM = 2 * Q_TILE + 4 * KV_STAGE + 1024;
    static constexpr int TM_S = KVB, TM_O = HD;                // TMEM columns of a tile
    // products of alternate blocks in places of their own where TMEM has them: they are added after the next weights are out
    // (4096 tokens, 64 heads of 64, f32: 340 us, with one place 361)
    static constexpr int O_BUF = SPLIT && 2 * KVB + 4 * HD <= 512 ? 2 : 1;
    static constexpr int CH = SPLIT ? 16 : 32;                 // positions whose weights lie together in TMEM
    // registers of the softmax warps, of the others: two warpgroups of each out of 512 x 128; launch_many checks that the
    // block starts with as many (a setmaxnreg.inc beyond them would wait forever)
    static constexpr int REG_SOFTMAX = SPLIT ? 192 : 176, REG_OTHER = 256 - REG_SOFTMAX;
};

__device__ __forceinline__ float kp_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// N (16 or 32) consecutive columns of this thread's TMEM lane: the load's start, and the wait that makes r readable
#define KP_R16(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), \
                     "=r"(r[o + 6]), "=r"(r[o + 7]), "=r"(r[o + 8]), "=r"(r[o + 9]), "=r"(r[o + 10]), "=r"(r[o + 11]), \
                     "=r"(r[o + 12]), "=r"(r[o + 13]), "=r"(r[o + 14]), "=r"(r[o + 15])
#define KP_RW16(r, o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), \
                      "+r"(r[o + 6]), "+r"(r[o + 7]), "+r"(r[o + 8]), "+r"(r[o + 9]), "+r"(r[o + 10]), "+r"(r[o + 11]), \
                      "+r"(r[o + 12]), "+r"(r[o + 13]), "+r"(r[o + 14]), "+r"(r[o + 15])
template <int N>
__device__ __forceinline__ void tmem_ld_start(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 16) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : KP_R16(r, 0) : "r"(taddr) : "memory");
    } else {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
                     "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                     : KP_R16(r, 0), KP_R16(r, 16) : "r"(taddr) : "memory");
    }
}
template <int N>
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[N]) {
    if constexpr (N == 16) asm volatile("tcgen05.wait::ld.sync.aligned;" : KP_RW16(r, 0)::"memory");
    else asm volatile("tcgen05.wait::ld.sync.aligned;" : KP_RW16(r, 0), KP_RW16(r, 16)::"memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t v[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t v[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[N]) {
    if constexpr (N == 8) tmem_st8(taddr, v);
    else if constexpr (N == 16) tmem_st16(taddr, v);
    else tmem_st32(taddr, v);
}
// mbar_wait of a whole warp, whose polls may sleep in the hardware: the other roles need the issue slots.  The lanes are
// together again on return, with one answer (tcgen05 instructions and elections need the whole warp).
__device__ __forceinline__ bool kp_wait(uint64_t *bar, uint32_t parity) {
    uint32_t done = 0;
    for (uint32_t i = 0; i < MBAR_POLLS && !done; i++)
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done) : "r"(smem_u32(bar)), "r"(parity), "r"(1000u) : "memory");
    return __all_sync(0xffffffffu, done);
}
// MMAs and commits issued by one elected lane of a converged warp: descriptors stay in uniform registers (from one
// divergent lane each MMA cost some 100 cycles of moves)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
                 "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar)) : "memory");
}
// V, [position][64 dimensions] rows of 128 bytes, 128-byte swizzle, dimensions contiguous ("MN-major"): 8-position
// groups 1024 bytes apart, planes of 64 dimensions `plane` bytes apart
__device__ __forceinline__ uint64_t desc_v(uint32_t addr, uint32_t plane) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(plane >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint32_t kp_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void kp_split(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h), r = fma2(f, make_float2(-1.f, -1.f), make_float2(a, b));
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = kp_h2(r.x, r.y);
}
__device__ __forceinline__ uint32_t kp_scale(uint32_t w, int b) { return __byte_perm(w, 0u, (b << 12) | (b << 4) | 0x404); }
__device__ __forceinline__ uint4 kp_eight(uint32_t codes, uint32_t f) {  // eight codes -> f16
    uint32_t h[4];
    e2m1x8_to_h2(codes, h);
    return make_uint4(hmul2_u32(h[0], f), hmul2_u32(h[1], f), hmul2_u32(h[2], f), hmul2_u32(h[3], f));
}

// One warp's 16-byte pieces of a block's keys or values, a phase at a time.
// KVB / 32 cache tiles have HD / 32 pieces each of keys, and of values.
template <int HD, int KVB>
struct KpPieces {
    static constexpr int PER = HD / 32, N = KVB / 32 * PER, MINE = (N + KP_DEQ - 1) / KP_DEQ;
    uint4 raw[MINE];
    uint32_t sc[MINE];
};

// What all blocks (and the join) agree on, from the sequences' lengths; a
// block's threads together.  Sequences with the most work first and pieces by
// the call's own length, not by the host's hint: three sequences of 5k to 16k
// 512 us, in their own order 595.
//   chunk  blocks of positions of a piece: a share of a block that fits the GPU
//          and a quarter more, so that units of one length stay whole and long
//          ones among short ones do not
//   order  the sequences, those with the most work first (up to KP_ORDER of them)
constexpr int KP_MIN = 6, KP_ORDER = 512;
struct KpPlan {
    long long part[KP_THREADS / 32];
    int cost[KP_ORDER];
    uint16_t order[KP_ORDER];
    int chunk;
    bool ordered;
};
template <int KVB>
__device__ __forceinline__ void kp_plan(KpPlan &p, const Kv4AttnArgs &a, int slots, int cuts) {
    const int n = a.c.n_seqs;
    const bool ordered = n > 1 && n <= KP_ORDER;
    long long sum = 0;
    if (ordered || cuts > 1) {
        for (int s = threadIdx.x; s < n; s += blockDim.x) {
            Kv4Seq q;
            q.load(a, s);
            const int c = q.nq > 0 ? (q.nq * a.gq + KP_ROWS - 1) / KP_ROWS * ((q.len - (q.first & ~31) + KVB - 1) / KVB) : 0;
            if (ordered) p.cost[s] = c;
            sum += (long long)c * a.c.n_kv;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) p.part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (ordered)
        for (int s = threadIdx.x; s < n; s += blockDim.x) {
            int r = 0;
            for (int k = 0; k < n; k++) r += p.cost[k] > p.cost[s] || (p.cost[k] == p.cost[s] && k < s);
            p.order[r] = (uint16_t)s;
        }
    if (threadIdx.x == 0) {
        sum = 0;
        for (int w = 0; w < (int)blockDim.x / 32; w++) sum += p.part[w];
        p.ordered = ordered;
        p.chunk = cuts > 1 ? (int)max((long long)KP_MIN * 128 / KVB, (sum * 5 / 4 + slots - 1) / slots) : 1 << 30;
    }
    __syncthreads();
}

// What a block does.  Each role works it out for itself after it has its
// registers: values that live across setmaxnreg are held to the smaller count
// and spilled (measured: the softmax twice as slow).
template <int KVB>
struct KpUnit {
    Kv4Seq q;
    int seq, kh, rt, rows, cut, ncut;  // rows from this block's first to the sequence's last
    int nblk, pos0;                    // blocks of positions of this piece, its first position
    int nb[2], first_p[2], last_p[2];  // per tile: blocks it needs, position of its first and last row
    // u: units (the sequences in order, later rows first: they see the most) x pieces, a unit's side by side; a unit has
    // as many of its `cuts` as pieces of about `chunk` blocks take
    __device__ __forceinline__ bool load(const Kv4AttnArgs &a, const KpPlan &p, int u, int row_tiles, int cuts) {
        cut = u % cuts;
        u /= cuts;
        kh = u % a.c.n_kv;
        u /= a.c.n_kv;
        rt = row_tiles - 1 - u % row_tiles;
        seq = u / row_tiles;
        if (p.ordered) seq = p.order[seq];
        q.load(a, seq);
        rows = q.nq * a.gq - rt * KP_ROWS;
        if (rows <= 0) return false;
        const int start = a.window > 0 ? (int)max(0LL, (long long)q.before + rt * KP_ROWS / a.gq - a.window + 1) & ~31 : 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r0 = rt * KP_ROWS + 128 * i, r1 = min(r0 + 127, q.nq * a.gq - 1);
            first_p[i] = q.before + r0 / a.gq;
            last_p[i] = q.before + r1 / a.gq;
            nb[i] = 128 * i < rows ? max(0, (last_p[i] + 1 - start + KVB - 1) / KVB) : 0;
        }
        const int all = max(nb[0], nb[1]);
        ncut = max(1, min(cuts, (int)(((long long)all + p.chunk - 1) / p.chunk)));
        if (cut >= ncut) return false;
        const int b0 = (int)((long long)all * cut / ncut), b1 = (int)((long long)all * (cut + 1) / ncut);
        nblk = b1 - b0;
        pos0 = start + b0 * KVB;
#pragma unroll
        for (int i = 0; i < 2; i++) nb[i] = max(0, min(nb[i], b1) - b0);
        return true;
    }
};

template <int HD, bool SPLIT, typename T>
__global__ void __launch_bounds__(KP_THREADS, 1) k_kv4_attn_many(Kv4AttnArgs a, int row_tiles, int cuts, int slots, int part_rows) {
    using C = KpCfg<HD, SPLIT>;
    constexpr int KVB = C::KVB, TB = kv4_tile_bytes(HD), G = HD / 32;
    extern __shared__ uint8_t raw_smem[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~(uintptr_t)1023);
    uint8_t *sq = base, *sk = base + 2 * C::Q_TILE, *sv = sk + 2 * C::KV_STAGE;
    __shared__ uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_half[2], p_full[2], o_full[2], q_full;
    __shared__ uint32_t tmem_base;
    __shared__ float s_factor[KP_ROWS];
    __shared__ int s_place;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    __shared__ KpPlan plan;
    kp_plan<KVB>(plan, a, slots, cuts);
    {
        KpUnit<KVB> u;
        if (!u.load(a, plan, blockIdx.x, row_tiles, cuts)) return;  // the whole block
        // a piece's long sums rest where its result goes; a call that cuts nothing leaves those places free, one per SM
        if (tid == 0) s_place = cuts > 1 ? (int)blockIdx.x : !SPLIT && u.nblk > KP_RUN ? kv4_take_place(a, KP_PLACE_ERR) : -1;
    }
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_full[i], KP_DEQ);
            mbar_init(&v_full[i], KP_DEQ);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_half[i], 4);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(&q_full, 8);
        fence_mbar_init();
    }
    if (warp == 15) tmem_alloc(&tmem_base, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_OTHER) : "memory");
        const uint32_t tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t *>(&tmem_base), 0);
        KpUnit<KVB> u;
        u.load(a, plan, blockIdx.x, row_tiles, cuts);
        const Kv4Seq &q = u.q;
        const int nblk = u.nblk, pos0 = u.pos0, seq = u.seq, kh = u.kh;
        bool ok = true;
        if (warp == 15) {
            // ------------------------------------------------ MMA issuer
            if (nblk > 0) {
                constexpr uint32_t id_s = umma_idesc_f16(128, KVB);
                constexpr uint32_t id_o = umma_idesc_f16(128, HD) | (1u << 16);  // B with its N contiguous
                // descriptors of the tiles' starts; an offset adds its sixteenth
                const uint64_t q_desc = umma_desc_sw128(smem_u32(sq)), k_desc = umma_desc_sw128(smem_u32(sk));
                const uint64_t v_desc = desc_v(smem_u32(sv), KVB * 128);
                auto scores = [&](int i, int b) {
                    const uint64_t qd = q_desc + (uint32_t)(i * C::Q_TILE / 16), kd = k_desc + (uint32_t)((b & 1) * C::KV_STAGE / 16);
                    const uint32_t d = tmem + i * C::TM_S;
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const int ko = (k >> 2) * (KVB * 128) + (k & 3) * 32, qo = (k >> 2) * (128 * 128) + (k & 3) * 32;
                        mma_ss(d, qd + qo / 16, kd + ko / 16, id_s, k > 0);
                        if (SPLIT) mma_ss(d, qd + (C::Q_HALF + qo) / 16, kd + ko / 16, id_s, 1u);
                    }
                    mma_commit(&s_full[i]);
                };
                auto products = [&](int i, int b, int half) {  // of the first or last positions of a block
                    const uint64_t vd = v_desc + (uint32_t)((b & 1) * C::KV_STAGE / 16);
                    const uint32_t o = tmem + 2 * C::TM_S + (i * C::O_BUF + (b & (C::O_BUF - 1))) * C::TM_O, p = tmem + i * C::TM_S;
#pragma unroll
                    for (int kk = 0; kk < KVB / 32; kk++) {
                        const int k = half * (KVB / 32) + kk;
                        // weights of CH positions: CH / 2 columns of hi, then of lo
                        const int at = k * 16 / C::CH * C::CH + k * 16 % C::CH / 2;
                        mma_ts(o, p + at, vd + k * 2048 / 16, id_o, k > 0 || (!SPLIT && (b & (KP_RUN - 1)) > 0));
                        if (SPLIT) mma_ts(o, p + at + C::CH / 2, vd + k * 2048 / 16, id_o, 1u);
                    }
                };
                ok = kp_wait(&q_full, 0) && kp_wait(&k_full[0], 0);
                tc_fence_after();
                if (ok) {
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        if (u.nb[i] > 0) scores(i, 0);
                    mma_commit(&k_empty[0]);
                }
                for (int b = 0; b < nblk && ok; b++) {
                    ok = kp_wait(&v_full[b & 1], (b >> 1) & 1);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        if (b >= u.nb[i] || !ok) continue;
                        ok = kp_wait(&p_half[i], b & 1);
                        if (!ok) continue;
                        tc_fence_after();
                        products(i, b, 0);
                        ok = kp_wait(&p_full[i], b & 1);
                        if (!ok) continue;
                        tc_fence_after();
                        products(i, b, 1);
                        if (b + 1 < u.nb[i]) {
                            ok = kp_wait(&k_full[(b + 1) & 1], ((b + 1) >> 1) & 1);
                            if (ok) scores(i, b + 1);
                        } else {
                            mma_commit(&o_full[i]);
                        }
                    }
                    mma_commit(&v_empty[b & 1]);
                    if (b + 1 < nblk) mma_commit(&k_empty[(b + 1) & 1]);
                }
                if (!ok && lane == 0) atomicExch(a.err, KP_ERR);
            }
        } else {
            // ------------------------------------------------ codes -> f16
            using P = KpPieces<HD, KVB>;
            const int w = warp - 8, g = lane >> 2, t = lane & 3;
            const int ntile = (int)((a.c.cap - 1) >> 5);
            const uint8_t *addr = nullptr;  // lane i: the cache tile addr_base + i of this piece
            int addr_base = -64;
            P kp, vp;
            auto load = [&](P &p, int b, bool key) {
                if (b >= nblk) return;
                constexpr int TILES = KVB / 32;
                if (b * TILES >= addr_base + 32) {
                    addr_base = b * TILES;
                    addr = a.c.tile(seq, kh, min((pos0 >> 5) + addr_base + lane, ntile), TB);
                }
#pragma unroll
                for (int x = 0; x < P::MINE; x++) {
                    const int y = w + x * KP_DEQ;
                    if (y >= P::N) break;
                    const uint8_t *tb = reinterpret_cast<const uint8_t *>(__shfl_sync(
                        0xffffffffu, reinterpret_cast<uint64_t>(addr), b * TILES + y / P::PER - addr_base));
                    const int pc = y % P::PER, u = HD == 64 ? pc : pc >> 1;
                    p.raw[x] = __ldg(reinterpret_cast<const uint4 *>(tb + (key ? 0 : 16 * HD) + pc * 512 + lane * 16));
                    p.sc[x] = __ldg(reinterpret_cast<const uint32_t *>(
                        tb + (key ? 32 * HD + (g * G + t * G / 4) * 4 : 33 * HD + ((t * G + g * G / 8) * 2 + u) * 4)));
                }
            };
            auto put = [&](uint8_t *stage, int row, int chunk, uint4 v) {
                *reinterpret_cast<uint4 *>(stage + (chunk >> 3) * (KVB * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) = v;
            };
            load(kp, 0, true);
            load(vp, 0, false);
            for (int b = 0; b < nblk && ok; b++) {
                const int st = b & 1;
                if (b >= 2) ok = kp_wait(&k_empty[st], ((b >> 1) - 1) & 1);
                if (!ok) break;
                uint8_t *ks = sk + st * C::KV_STAGE, *vs = sv + st * C::KV_STAGE;
#pragma unroll
                for (int x = 0; x < P::MINE; x++) {
                    const int y = w + x * KP_DEQ;
                    if (y >= P::N) break;
                    const int row0 = y / P::PER * 32, pc = y % P::PER;
                    const uint32_t *cw = reinterpret_cast<const uint32_t *>(&kp.raw[x]);
                    if constexpr (HD == 64) {  // words: position 2 g + (0, 1) x 16 dimensions
                        const int odd = g & 1;  // odd lanes take the other half first: no two lanes on a bank
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const uint32_t f = kp_scale(kp.sc[x], 2 * pc + j);
                            const int row = row0 + 16 * pc + 2 * g + j;
                            const uint32_t c0 = odd ? cw[2 * j + 1] : cw[2 * j], c1 = odd ? cw[2 * j] : cw[2 * j + 1];
                            put(ks, row, 2 * t + odd, kp_eight(c0, f));
                            put(ks, row, 2 * t + (odd ^ 1), kp_eight(c1, f));
                        }
                    } else {  // words: 32 dimensions of position 2 g + j
                        const int far = t >> 1;
                        const uint32_t f = __byte_perm(kp.sc[x], 0u, (pc << 12) | (pc << 4) | 0x404);
                        const int row = row0 + 16 * (pc >> 1) + 2 * g + (pc & 1);
#pragma unroll
                        for (int k = 0; k < 4; k += 2) {
                            const uint32_t c0 = far ? cw[k + 1] : cw[k], c1 = far ? cw[k] : cw[k + 1];
                            put(ks, row, 4 * t + k + far, kp_eight(c0, f));
                            put(ks, row, 4 * t + k + (far ^ 1), kp_eight(c1, f));
                        }
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[st]);
                load(kp, b + 1, true);

                if (b >= 2) ok = kp_wait(&v_empty[st], ((b >> 1) - 1) & 1);
                if (!ok) break;
                const int bp = pos0 + b * KVB;
#pragma unroll
                for (int x = 0; x < P::MINE; x++) {
                    const int y = w + x * KP_DEQ;
                    if (y >= P::N) break;
                    const int row0 = y / P::PER * 32, pc = y % P::PER, u = HD == 64 ? pc : pc >> 1;
                    const uint32_t *cw = reinterpret_cast<const uint32_t *>(&vp.raw[x]);
                    uint32_t sc = vp.sc[x];
                    {   // positions that nobody wrote: any byte may stand there, a NaN scale among them
                        const int p = bp + row0 + 16 * u + 4 * t, above = q.len - p, below = q.first - p;
                        if (above < 4) sc &= above <= 0 ? 0u : (1u << (8 * above)) - 1u;
                        if (below > 0) sc &= below >= 4 ? 0u : ~((1u << (8 * below)) - 1u);
                    }
                    const int far = t >> 1;
                    if constexpr (HD == 64) {  // words: 8 dimensions of position 4 t + i
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int ii = i ^ (far << 1);
                            const uint32_t c = far ? cw[i ^ 2] : cw[i];
                            put(vs, row0 + 16 * u + 4 * t + ii, g, kp_eight(c, __byte_perm(sc, 0u, (ii << 12) | (ii << 4) | 0x404)));
                        }
                    } else {  // words: 16 dimensions of position 4 t + c, then of 4 t + c + 2
#pragma unroll
                        for (int s = 0; s < 2; s++) {
                            const int i = (pc & 1) + 2 * s;
                            const uint32_t f = __byte_perm(sc, 0u, (i << 12) | (i << 4) | 0x404);
                            const int row = row0 + 16 * u + 4 * t + i;
                            const uint32_t c0 = far ? cw[2 * s + 1] : cw[2 * s], c1 = far ? cw[2 * s] : cw[2 * s + 1];
                            put(vs, row, 2 * g + far, kp_eight(c0, f));
                            put(vs, row, 2 * g + (far ^ 1), kp_eight(c1, f));
                        }
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
                load(vp, b + 1, false);
            }
            if (!ok && lane == 0) atomicExch(a.err, KP_ERR);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_SOFTMAX) : "memory");
        const uint32_t tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t *>(&tmem_base), 0);
        KpUnit<KVB> u;
        u.load(a, plan, blockIdx.x, row_tiles, cuts);
        const Kv4Seq &q = u.q;
        const int rt = u.rt, kh = u.kh, ncut = u.ncut, pos0 = u.pos0, before = q.before;
        bool ok = true;
        // ---------------------------------------------------- softmax, thread = row
        const int i = warp >> 2, blocks = i ? u.nb[1] : u.nb[0];
        const int first_row_p = i ? u.first_p[1] : u.first_p[0], last_row_p = i ? u.last_p[1] : u.last_p[0];
        const int r = tid & 127, row = rt * KP_ROWS + 128 * i + r;
        const int j = row / a.gq, h = kh * a.gq + row - j * a.gq;
        const bool live = j < q.nq;
        const int hi = live ? before + j : -1, lo = a.window > 0 ? max(0, hi - a.window + 1) : 0;
        {   // the queries, scaled to below 2 by a power of two per row, into the swizzled tile; the scale's sign goes with
            // them.  A row takes HD / 8 lanes, a lane one 16-byte chunk of the tile.
            constexpr int L = HD / 8, STEP = 32 / L, N = 32 / STEP;
            const int first = 32 * (warp & 3), c = lane % L;
            float x[N][8];
#pragma unroll
            for (int k = 0; k < N; k++) {
                const int rr = rt * KP_ROWS + 128 * i + first + k * STEP + lane / L, jj = rr / a.gq;
                if (jj < q.nq) {
                    load_row<8>(static_cast<const T *>(a.q) + (int64_t)(q.q0 + jj) * a.ldq +
                                    (int64_t)(kh * a.gq + rr - jj * a.gq) * HD + 8 * c, a.q_wide, x[k]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[k][e] = 0.f;
                }
                if (SPLIT && HD == 128 && k % 8 == 7) asm volatile("" ::: "memory");  // eight rows' loads at a time
            }
#pragma unroll
            for (int k = 0; k < N; k++) {
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[k][e]));
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
                const float down = __uint_as_float((254u - e) << 23) * (a.scale < 0.f ? -1.f : 1.f);
                uint32_t vh[4], vl[4];
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    if (SPLIT) kp_split(x[k][2 * y] * down, x[k][2 * y + 1] * down, vh[y], vl[y]);
                    else vh[y] = kp_h2(x[k][2 * y] * down, x[k][2 * y + 1] * down);
                }
                const int rr = first + k * STEP + lane / L;
                uint8_t *at = sq + i * C::Q_TILE + rr * 128 + (c >> 3) * (128 * 128) + (((c & 7) ^ (rr & 7)) << 4);
                *reinterpret_cast<uint4 *>(at) = make_uint4(vh[0], vh[1], vh[2], vh[3]);
                if (SPLIT) *reinterpret_cast<uint4 *>(at + C::Q_HALF) = make_uint4(vl[0], vl[1], vl[2], vl[3]);
                if (c == 0) s_factor[128 * i + rr] = fabsf(a.scale) * LOG2E * __uint_as_float(e << 23);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
        }
        const float factor = fmaxf(s_factor[128 * i + r], 1e-37f);  // above zero: a masked -infinity times it stays one
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + i * C::TM_S, to = tmem + lanes + 2 * C::TM_S + i * C::O_BUF * C::TM_O;
        float m = -INFINITY, l = 0.f;
        float o[HD];
        // the weights stored so far are P's (or its first half's)
        auto weights_out = [&](uint64_t *bar) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        if constexpr (SPLIT) {
            // f32: O in registers, each block's product added with the factor that its maximum gave
            float alpha = 1.f;
#pragma unroll
            for (int k = 0; k < HD; k++) o[k] = 0.f;
            constexpr int CH = C::CH, NC = KVB / CH;
            uint32_t ra[CH], rb[CH];
            // a block's columns of this lane, `f` called with each CH of them while the next ones load.  Blocks that every
            // row sees whole take straight-line code: a branch costs some 50 cycles here (the roles' code is far apart)
            auto columns = [&](auto edge, auto &&f) {
                constexpr int U = decltype(edge)::value ? 1 : NC / 2;
                tmem_ld_start(ts, ra);
#pragma unroll U
                for (int c = 0; c < NC; c += 2) {
                    tmem_ld_wait(ra);
                    tmem_ld_start(ts + CH * (c + 1), rb);
                    f(c, ra);
                    tmem_ld_wait(rb);
                    if (c + 2 < NC) tmem_ld_start(ts + CH * (c + 2), ra);
                    f(c + 1, rb);
                }
            };
            auto add_products = [&](int b, float alpha) {  // block b's, with the factor that its maximum gave
                const uint32_t at = to + (b & (C::O_BUF - 1)) * C::TM_O;
                auto add = [&](int k, uint32_t x, uint32_t y) {
                    const float2 v = fma2(make_float2(o[k], o[k + 1]), make_float2(alpha, alpha),
                                          make_float2(__uint_as_float(x), __uint_as_float(y)));
                    o[k] = v.x;
                    o[k + 1] = v.y;
                };
                tmem_ld_start(at, ra);
#pragma unroll
                for (int c = 0; c < HD / CH; c += 2) {
                    tmem_ld_wait(ra);
                    tmem_ld_start(at + CH * (c + 1), rb);
#pragma unroll
                    for (int k = 0; k < CH; k += 2) add(CH * c + k, ra[k], ra[k + 1]);
                    tmem_ld_wait(rb);
                    if (c + 2 < HD / CH) tmem_ld_start(at + CH * (c + 2), ra);
#pragma unroll
                    for (int k = 0; k < CH; k += 2) add(CH * (c + 1) + k, rb[k], rb[k + 1]);
                }
            };
            for (int b = 0; b < blocks; b++) {
                ok = kp_wait(&s_full[i], b & 1);  // implies that the block before's products are complete
                if (!ok) break;
                tc_fence_after();
                if (C::O_BUF == 1 && b > 0) add_products(b - 1, alpha);
                const float last = alpha;
                const int bp = pos0 + b * KVB;
                float2 sum = make_float2(0.f, 0.f);
                auto block = [&](auto edge) {
                    constexpr bool EDGE = decltype(edge)::value;
                    float top = -INFINITY;
                    columns(edge, [&](int c, uint32_t (&r)[CH]) {
                        if (EDGE) {
                            const int up = hi - bp - CH * c, down = lo - bp - CH * c;
#pragma unroll
                            for (int k = 0; k < CH; k++) r[k] = k <= up && k >= down ? r[k] : 0xff800000u;
                        }
                        float t4[4];
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            t4[k] = max3(__uint_as_float(r[k]), __uint_as_float(r[k + 4]), __uint_as_float(r[k + 8]));
#pragma unroll
                        for (int k = 0; k < 4; k += 2) t4[k] = max3(t4[k], __uint_as_float(r[12 + k]), __uint_as_float(r[13 + k]));
                        top = max3(top, max3(t4[0], t4[1], t4[2]), t4[3]);
                    });
                    const float mn = top == -INFINITY ? m : fmaxf(m, __fmaf_ru(top, factor, -KV4_AHEAD));
                    const float mm = mn == -INFINITY ? 0.f : mn;
                    alpha = kp_ex2(m - mm);
                    m = mn;
                    columns(edge, [&](int c, uint32_t (&r)[CH]) {
                        uint32_t w[CH];
                        float e[CH];
#pragma unroll
                        for (int k = 0; k < CH; k += 2) {
                            const float2 x = fma2(make_float2(__uint_as_float(r[k]), __uint_as_float(r[k + 1])),
                                                  make_float2(factor, factor), make_float2(-mm, -mm));
                            e[k] = kp_ex2(x.x);
                            e[k + 1] = kp_ex2(x.y);
                        }
                        if (EDGE) {
                            const int up = hi - bp - CH * c, down = lo - bp - CH * c;
#pragma unroll
                            for (int k = 0; k < CH; k++) e[k] = k <= up && k >= down ? e[k] : 0.f;
                        }
#pragma unroll
                        for (int k = 0; k < CH; k += 2) {
                            sum = add2(sum, make_float2(e[k], e[k + 1]));
                            kp_split(e[k], e[k + 1], w[k / 2], w[CH / 2 + k / 2]);
                        }
                        tmem_st(ts + CH * c, w);
                        if (c == NC / 2 - 1) weights_out(&p_half[i]);
                    });
                };
                // some row does not see some position of the block
                if (bp + KVB - 1 > first_row_p || (a.window > 0 && bp <= last_row_p - a.window)) block(std::true_type{});
                else block(std::false_type{});
                l = fmaf(l, alpha, sum.x + sum.y);
                weights_out(&p_full[i]);
                if (C::O_BUF == 2 && b > 0) add_products(b - 1, last);
            }
            if (blocks > 0 && ok) {
                ok = kp_wait(&o_full[i], 0);
                tc_fence_after();
                if (ok) add_products(blocks - 1, alpha);
            }
        } else {
            // f16, bf16: O stays in TMEM; m is followed up, and O and l rescaled, only when the largest x is more than KV4_LAG
            // above the one that m was taken from (weights of up to 2^15 all the same).
            // The tensor core truncates its running sum, some 2^-22.5 of it with each MMA: values of one sign lose 5.4e-9 of
            // theirs a position (measured: 7e-4 of 131072).  So after KP_RUN blocks O goes to the row's place in memory,
            // against `rest_m`, and the next products start from zero.
            float rest_m = -INFINITY;
            // (a warp's rows share the part that its results go to in the end, four columns of each side by side)
            const int near = min(32, part_rows - (128 * i + (r & ~31)));
            auto place = [&](int c) {
                return a.parts + (size_t)s_place * part_rows * (HD + 2) + 2 * part_rows + (128 * i + (r & ~31)) * HD +
                       c * near + lane * 4;
            };
            auto add_rest = [&](float *x, int c, float f) {  // columns c .. c + 31 of what rests, times f
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(place(c + k)));
                    x[k] = fmaf(v.x, f, x[k]);
                    x[k + 1] = fmaf(v.y, f, x[k + 1]);
                    x[k + 2] = fmaf(v.z, f, x[k + 2]);
                    x[k + 3] = fmaf(v.w, f, x[k + 3]);
                }
            };
            auto rest_factor = [&] { return m == -INFINITY ? 0.f : kp_ex2(rest_m - m); };
            auto put_to_rest = [&](bool first) {  // O, whose products are complete
                const float f = rest_factor();
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t v[32];
                    tmem_ld_start(to + c, v);
                    tmem_ld_wait(v);
                    float x[32];
#pragma unroll
                    for (int k = 0; k < 32; k++) x[k] = __uint_as_float(v[k]);
                    if (live) {
                        if (!first) add_rest(x, c, f);
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            __stcg(reinterpret_cast<float4 *>(place(c + k)), make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]));
                    }
                    __syncwarp();
                }
                rest_m = m;
            };
            for (int b = 0, run = 0; b < blocks && ok; run = b) {
                if (run > 0) {
                    ok = kp_wait(&s_full[i], b & 1);
                    if (!ok) break;
                    tc_fence_after();
                    put_to_rest(run == KP_RUN);
                }
                const int end = min(blocks, run + KP_RUN);
                for (; b < end; b++) {
                    ok = kp_wait(&s_full[i], b & 1);  // implies that the block before's products are complete
                    if (!ok) break;
                    tc_fence_after();
                    uint32_t r[KVB / 32][32];
#pragma unroll
                    for (int c = 0; c < KVB / 32; c++) tmem_ld_start(ts + 32 * c, r[c]);
#pragma unroll
                    for (int c = 0; c < KVB / 32; c++) tmem_ld_wait(r[c]);
                    const int bp = pos0 + b * KVB;
                    // some row does not see some position of the block
                    if (bp + KVB - 1 > first_row_p || (a.window > 0 && bp <= last_row_p - a.window)) {
                        const int up = hi - bp, down = lo - bp;
#pragma unroll
                        for (int k = 0; k < KVB; k++) r[k / 32][k % 32] = k <= up && k >= down ? r[k / 32][k % 32] : 0xff800000u;
                    }
                    float t4[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        t4[c] = -INFINITY;
#pragma unroll
                        for (int k = 0; k < 32; k += 2) t4[c] = max3(t4[c], __uint_as_float(r[c][k]), __uint_as_float(r[c][k + 1]));
                    }
                    const float top = max3(fmaxf(t4[0], t4[1]), t4[2], t4[3]);
                    const float need = top == -INFINITY ? -INFINITY : __fmaf_ru(top, factor, KV4_LAG - KV4_AHEAD);
                    if (__any_sync(0xffffffffu, need - m > KV4_LAG)) {  // m = -infinity: any number
                        const float mn = fmaxf(m, need), alpha = mn == -INFINITY ? 1.f : kp_ex2(m - mn);
                        m = mn;
                        l *= alpha;
                        if (b > run) {
#pragma unroll 1
                            for (int c = 0; c < HD; c += 16) {
                                uint32_t v[16];
                                tmem_ld_start(to + c, v);
                                tmem_ld_wait(v);
#pragma unroll
                                for (int k = 0; k < 16; k++) v[k] = __float_as_uint(__uint_as_float(v[k]) * alpha);
                                tmem_st(to + c, v);
                            }
                        }
                    }
                    const float mm = m == -INFINITY ? 0.f : m;
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < KVB / 32; c++) {
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            const float2 x = fma2(make_float2(__uint_as_float(r[c][k]), __uint_as_float(r[c][k + 1])),
                                                  make_float2(factor, factor), make_float2(-mm, -mm));
                            const float2 e = make_float2(kp_ex2(x.x), kp_ex2(x.y));
                            sum[k / 2 % 2] = add2(sum[k / 2 % 2], e);
                            w[k / 2] = kp_h2(e.x, e.y);
                        }
                        tmem_st(ts + 32 * c, w);
                        if (c == KVB / 64 - 1) weights_out(&p_half[i]);
                    }
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    weights_out(&p_full[i]);
                }
            }
#pragma unroll
            for (int k = 0; k < HD; k++) o[k] = 0.f;
            if (blocks > 0 && ok) {
                ok = kp_wait(&o_full[i], 0);
                tc_fence_after();
                if (ok) {
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t v[32];
                        tmem_ld_start(to + c, v);
                        tmem_ld_wait(v);
#pragma unroll
                        for (int k = 0; k < 32; k++) o[c + k] = __uint_as_float(v[k]);
                    }
                    if (blocks > KP_RUN && live) {
                        const float f = rest_factor();
#pragma unroll
                        for (int c = 0; c < HD; c += 32) add_rest(o + c, c, f);
                    }
                    __syncwarp();  // all have read: a piece's results may go there
                }
            }
        }
        if (!ok && lane == 0) atomicExch(a.err, KP_ERR);
        // ---- the row's result, or this piece's part of it
        const float sk2 = a.sinks && live ? a.sinks[h] * LOG2E : -INFINITY;
        if (ncut == 1) {
            if (live) {
                const float M = fmaxf(m, sk2), mm = M == -INFINITY ? 0.f : M, e = kp_ex2(m - mm);
                const float L = l * e + (a.sinks ? kp_ex2(sk2 - mm) : 0.f), f = L > 0.f ? e / L : 0.f;
                T *dst = static_cast<T *>(a.out) + (int64_t)(q.q0 + j) * a.ldo + (int64_t)h * HD;
#pragma unroll
                for (int k = 0; k < HD; k += 4)
                    store4f(dst + k, a.out_wide, make_float4(o[k] * f, o[k + 1] * f, o[k + 2] * f, o[k + 3] * f));
            }
        } else {
            // for k_kv4_join
            if (live) {
                float *part = a.parts + (size_t)blockIdx.x * part_rows * (HD + 2);
                const int rr = 128 * i + r;
                part[rr] = m;
                part[part_rows + rr] = l;
#pragma unroll
                for (int k = 0; k < HD; k += 4)
                    *reinterpret_cast<float4 *>(part + 2 * part_rows + (size_t)rr * HD + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 15) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
    if (cuts == 1 && tid == 0 && s_place >= 0) kv4_leave_place(a, s_place);
}

template <int N> __device__ __forceinline__ void load_f(const float *src, float v[N]) {
    if constexpr (N == 4) {
        const float4 x = __ldg(reinterpret_cast<const float4 *>(src));
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
        const float2 x = __ldg(reinterpret_cast<const float2 *>(src));
        v[0] = x.x; v[1] = x.y;
    }
}

// The pieces of cut units joined: a warp a row, HD / 32 outputs a lane, in
// piece order.  Bound: the pieces' bytes from L2 (a launch's 2 to 4 us); in
// the last piece to finish, as the few-row kernel joins, one block would read
// 256 rows of every piece.
constexpr int KJ_WARPS = 8;
template <int HD, int KVB, typename T>
__global__ void __launch_bounds__(KJ_WARPS * 32) k_kv4_join(Kv4AttnArgs a, int row_tiles, int cuts, int slots, int part_rows) {
    constexpr int N = HD / 32;
    __shared__ KpPlan plan;
    kp_plan<KVB>(plan, a, slots, cuts);
    const int per = (part_rows + KJ_WARPS - 1) / KJ_WARPS, unit = blockIdx.x / per, lane = threadIdx.x & 31;
    const int r = (blockIdx.x % per) * KJ_WARPS + (threadIdx.x >> 5);
    KpUnit<KVB> u;
    if (!u.load(a, plan, unit * cuts, row_tiles, cuts) || u.ncut == 1) return;
    if (r >= min(u.rows, part_rows)) return;
    const int row = u.rt * KP_ROWS + r, j = row / a.gq, h = u.kh * a.gq + row - j * a.gq;
    const size_t PF = (size_t)part_rows * (HD + 2);
    const float *parts = a.parts + (size_t)unit * cuts * PF;
    const float sk = a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
    float M = sk;
    for (int c = lane; c < u.ncut; c += 32) M = fmaxf(M, __ldg(parts + c * PF + r));
    M = warp_max(M);
    const float mm = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc[N];
#pragma unroll
    for (int k = 0; k < N; k++) acc[k] = 0.f;
#pragma unroll 4
    for (int c = 0; c < u.ncut; c++) {
        const float *p = parts + c * PF, e = kp_ex2(__ldg(p + r) - mm);
        const float *src = p + 2 * part_rows + (size_t)r * HD + lane * N;
        L += __ldg(p + part_rows + r) * e;
        float v[N];
        load_f<N>(src, v);
#pragma unroll
        for (int k = 0; k < N; k++) acc[k] += v[k] * e;
    }
    L += a.sinks ? kp_ex2(sk - mm) : 0.f;
    const float f = L > 0.f ? 1.f / L : 0.f;
    T *dst = static_cast<T *>(a.out) + (int64_t)(u.q.q0 + j) * a.ldo + (int64_t)h * HD + lane * N;
#pragma unroll
    for (int k = 0; k < N; k++) dst[k] = from_f32<T>(acc[k] * f);
}

// How a call may be cut: units (sequence, key/value head, two row tiles) in
// as many pieces of KP_MIN x 128 positions or more as there are places for
// their results: the rows of one round of full blocks, and KP_ROUNDS rounds of
// blocks at most.  kp_plan says on the device how far it is.
constexpr int KP_ROUNDS = 3;
int64_t kv4_many_part_floats(int sms) { return (int64_t)sms * KP_ROWS * (128 + 2); }
struct ManyCut {
    int row_tiles, cuts, part_rows;
};
static ManyCut many_cut(const Kv4AttnArgs &a, int64_t max_kv) {
    ManyCut m;
    const int64_t rows = (int64_t)a.max_q * a.gq;
    m.row_tiles = ceil_div(rows, KP_ROWS);
    m.part_rows = (int)(rows < KP_ROWS ? (rows + 7) / 8 * 8 : KP_ROWS);
    int64_t len = a.window > 0 && max_kv > (int64_t)a.window + a.max_q ? (int64_t)a.window + a.max_q : max_kv;
    const int64_t blocks = len < 1 ? 1 : (len + 127) / 128, units = (int64_t)a.c.n_seqs * a.c.n_kv * m.row_tiles;
    int64_t pieces = (int64_t)num_sms() * KP_ROWS / m.part_rows;
    if (pieces > (int64_t)num_sms() * KP_ROUNDS) pieces = (int64_t)num_sms() * KP_ROUNDS;
    int64_t cuts = pieces / units, most = blocks / KP_MIN;
    if (cuts > most) cuts = most;
    m.cuts = (int)(cuts < 1 ? 1 : cuts);
    return m;
}

template <int HD, bool SPLIT, typename T>
static int launch_many(const Kv4AttnArgs &a, const ManyCut &m, cudaStream_t st) {
    using C = KpCfg<HD, SPLIT>;
    TRY(ensure_smem(k_kv4_attn_many<HD, SPLIT, T>, C::SMEM));
    static int regs = 0;  // of a thread at launch
    if (!regs) {
        cudaFuncAttributes f{};
        MG_CUDA(cudaFuncGetAttributes(&f, k_kv4_attn_many<HD, SPLIT, T>));
        regs = f.numRegs;
    }
    MG_REQUIRE(regs * KP_THREADS >= 256 * (C::REG_SOFTMAX + C::REG_OTHER), MG_ERR_CUDA,
               "kv4_attn: built with %d registers a thread, too few for its split", regs);
    const int64_t blocks = (int64_t)m.row_tiles * a.c.n_seqs * a.c.n_kv * m.cuts;
    MG_REQUIRE(blocks < (1LL << 31), MG_ERR_ARG, "kv4_attn: too many rows");
    k_kv4_attn_many<HD, SPLIT, T><<<(unsigned)blocks, KP_THREADS, C::SMEM, st>>>(a, m.row_tiles, m.cuts, num_sms(), m.part_rows);
    MG_CHECK_LAUNCH();
    if (m.cuts > 1) {
        const int64_t join = blocks / m.cuts * ceil_div(m.part_rows, KJ_WARPS);
        k_kv4_join<HD, C::KVB, T><<<(unsigned)join, KJ_WARPS * 32, 0, st>>>(a, m.row_tiles, m.cuts, num_sms(), m.part_rows);
        MG_CHECK_LAUNCH();
    }
    return MG_OK;
}

int kv4_attn_many(const Kv4AttnArgs &a, int hd, int act, int64_t max_kv, cudaStream_t st) {
    const ManyCut m = many_cut(a, max_kv);
    if (act == MG_ACT_F32)
        return hd == 64 ? launch_many<64, true, float>(a, m, st) : launch_many<128, true, float>(a, m, st);
    if (act == MG_ACT_F16)
        return hd == 64 ? launch_many<64, false, __half>(a, m, st) : launch_many<128, false, __half>(a, m, st);
    return hd == 64 ? launch_many<64, false, __nv_bfloat16>(a, m, st)
                    : launch_many<128, false, __nv_bfloat16>(a, m, st);
}

}  // namespace mg
