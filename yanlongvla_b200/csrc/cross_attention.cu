// Attention to an encoder's states of another length: out = softmax(scale q k^T) v over the states that are there.
//
// q (B S, T, heads D): the S batches b S .. b S + S - 1 read the states of sequence b; k, v (B, N, kv_heads D); lens (B) and a mask
// (B, N) say which states are there. The rows that read one key head of one sequence are its R = S T group queries, token by
// token, `group` heads to a token: they share every load of K and V.
#include "memory.cuh"
#include "tc.cuh"

__device__ int g_tcq_cross_error;

int tcq_cross_error(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tcq_cross_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && v) {
        const int z = 0;
        if (cudaMemcpyToSymbol(g_tcq_cross_error, &z, sizeof(int)) != cudaSuccess) return -1;
    }
    return v;
}

namespace {

using namespace tcq;

struct CrossArgs {
    const u16* q;
    i64 q_sb, q_st;
    u16* out;
    const int* lens;
    const unsigned char* mask;
    i64 mask_sb;
    int B, S, T, N, heads, kv_heads, group, D, rows;      // rows: S T group
    int kb, vb;                                           // 0: all sequences share one batch of keys, of values in memory
    FastDiv by_group, by_tokens;                          // tokens: T
    float scale_log2;                                     // scale * log2(e)
};

TCQ_HD int states_of(const CrossArgs& A, int b) {
    if (!A.lens) return A.N;
    const int n = A.lens[b];
    if ((unsigned)n > (unsigned)A.N) {
        atomicOr(&g_tcq_cross_error, 2);
        return n < 0 ? 0 : A.N;
    }
    return n;
}

// Element offset of row r of key head h, sequence b, in q (strides) or in out (contiguous).
TCQ_HD i64 row_at(const CrossArgs& A, int b, int h, int r, i64 sb, i64 st) {
    const int tok = (int)fdiv((unsigned)r, A.by_group), g = r - tok * A.group;
    const int s = (int)fdiv((unsigned)tok, A.by_tokens), t = tok - s * A.T;
    return ((i64)b * A.S + s) * sb + t * st + (i64)(h * A.group + g) * A.D;
}

__device__ __forceinline__ void tma_load_4d(u32 dst, const CUtensorMap* map, u32 bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

// Scores come as (q k) c with c > 0, so that their order is known before the scaling: a negative scale turns the queries, a scale of zero
// makes them zero.
TCQ_HD float score_scale(const CrossArgs& A) { return A.scale_log2 == 0.f ? 1.f : fabsf(A.scale_log2); }
TCQ_HD u32 query_flip(const CrossArgs& A) { return A.scale_log2 < 0.f ? 0x80008000u : 0u; }
TCQ_HD u32 query_keep(const CrossArgs& A) { return A.scale_log2 == 0.f ? 0u : ~0u; }

// Two weights or outputs, rounded to nearest even (a NaN of any kind stays one); lo in the low half.
template <int DT>
TCQ_HD u32 weights2(float lo, float hi) {
    u32 r;
    if (DT == TCQ_DT_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The factor of a part with reference ml.x and sum ml.y next to others of reference up to top: a part without weight adds nothing, unless
// its sum is NaN (scores that are NaN move no reference): the row has to say so.
TCQ_HD float part_factor(float2 ml, float top) { return top == -INFINITY ? (ml.y == ml.y ? 0.f : 1.f) : ml.y != ml.y ? 1.f : ex2(ml.x - top); }

// Weights are 2^(x - m + kRef), m the row's reference, moved only when a score passes it by more than kSlack: below 2^13, so
// that FP16 holds them with 11 bits from there down to 2^-14.
// The weights come of one fused step, s c + (kRef - m): m, and the difference, are off by half a step of FP32 at |m| each, one in the
// exponent together at 2^24. Past that the weights would leave the type's range, either way: a row whose reference ends there is
// reported. (Scores less their reference before the scaling are right at any size, but cost 4 to 13 %: 17 queries over 160 states
// 4.45 -> 4.83 us, 8 x 16 candidates 14.7 -> 16.7, 2 x 4096 x 4096 with heads of 128 514 -> 533.)
constexpr float kRef = 5.f, kSlack = 8.f, kMost = 16777216.f;
TCQ_HD bool past_range(float m) { return fabsf(m) > kMost && fabsf(m) != INFINITY; }

// ------------------------------------------------------------------------------------------------ products of 16 rows
// Warps of 16 query rows on m16n8k16 products, for few rows or few states: bound by HBM where the states are many, by latency where
// they are few. A CTA has four such warps and one that requests the states. WM of the warps take 16 rows each of one unit (the rows
// of a key head of a sequence, in blocks of 16 WM); the 4 / WM rings of states serve
//   - whole: a unit each (many units: nothing to add up), or
//   - the same unit, its states divided among the rings of a cluster's CTAs (few units). A row's parts are added in shared memory, a
//     cluster's through distributed shared memory, always in the same order.
// A ring holds chunks of 32 states (16 above head width 64): TMA, 128-byte swizzle, zeros past D and N. The requesting warp
// passes over chunks of which the mask leaves nothing, and tells what each stage holds. Up to head width 64 a warp takes two tiles of 16
// rows where there are more than 16 (fragments of K and V read once for both).
//
// One token of four sequences over 16411 states of 8 heads of 64: 26 us, 5.1 TB/s. 32 x 17 queries over 160 states, 32 heads of 48: 8.0 us
// (requests by the computing warps 24.5, by a warp ring after ring 15.6, by a lane for each ring 8.5), bound by five chunks in a
// row of 700 to 1,000 clocks in each of eight warps an SM, which 168 registers leave.
constexpr int kRowWarps = 4, kRowThreads = 32 * (kRowWarps + 1);

TCQ_HD void ldsm4(u32 addr, u32 (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
TCQ_HD void ldsm4t(u32 addr, u32 (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int DT>
TCQ_HD void mma16816(float (&d)[4], u32 a0, u32 a1, u32 a2, u32 a3, u32 b0, u32 b1) {
    if (DT == TCQ_DT_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Shared memory of a CTA: the rings, then their barriers and what each stage holds. Parts overlay the rings.
template <int DP, int MT>
struct Rows {
    static constexpr int CHUNK = DP <= 64 ? 32 : 16;                                                 // states
    static constexpr int ATOMS = (DP + 63) / 64, HALF = ATOMS * CHUNK * 128, STAGE = 2 * HALF;       // bytes of a chunk's keys, of both: 8 KB
    static constexpr int PITCH = DP + 4;                                                             // floats of a part's row
    static constexpr int ROWS = 16 * MT;                                                             // of a warp
    static constexpr int PARTS = kRowWarps * ROWS * PITCH * 4, ML = ROWS * kRowWarps * 8;               // parts, then m and l of the CTA's rows
    static constexpr int MOST = 6;                                                                   // stages of a ring, at most
    static constexpr int ring_bytes(int rings, int stages) {
        return rings * stages * STAGE > PARTS + ML ? rings * stages * STAGE : PARTS + ML;
    }
    static constexpr int bytes(int rings, int stages) { return ring_bytes(rings, stages) + rings * stages * 24 + 16; }
};
struct RowsPlan {
    int wm_log2, stages, splits, whole, row_blocks, block_rows, units;
    FastDiv by_blocks, by_heads, by_splits, by_workers;
};

template <int DT, int DP, int MT>
__global__ void __launch_bounds__(kRowThreads, MT == 2 ? 2 : DP <= 48 ? 4 : DP <= 64 ? 3 : 2)
k_cross_rows(const CrossArgs A, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const RowsPlan R) {
    typedef Rows<DP, MT> P;
    constexpr int KS = DP / 16, NT = DP / 8, NK = P::CHUNK / 8, RINGS = kRowWarps;
    constexpr u32 kAll = (u32)((1ull << P::CHUNK) - 1);
    extern __shared__ __align__(1024) char smem_rows[];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int WM = 1 << R.wm_log2, rings = kRowWarps >> R.wm_log2, wm = warp & (WM - 1), kg = warp >> R.wm_log2, stages = R.stages;
    const u32 sbase = smem_u32(smem_rows);
    const int ring_bytes = P::ring_bytes(rings, stages);
    const u32 bars = sbase + ring_bytes;                           // full, empty of each stage of each ring
    int2* meta = reinterpret_cast<int2*>(smem_rows + ring_bytes + rings * stages * 16);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_rows + ring_bytes + rings * stages * 24);
    if (tid < rings * stages) {
        mbar_init(bars + 16 * tid, 1);
        mbar_init(bars + 16 * tid + 8, WM);
        if (tid == 0) *abort_flag = 0;
        mbar_init_fence();
    }
    const int rank = (int)(blockIdx.x - fdiv(blockIdx.x, R.by_splits) * R.splits);
    // the unit of ring k: row block, sequence and key head
    auto unit_of = [&](int k, int& rb, int& b, int& h) {
        const int u = R.whole ? blockIdx.x * rings + k : (int)fdiv(blockIdx.x, R.by_splits);
        const int bh = (int)fdiv((unsigned)u, R.by_blocks);
        rb = u - bh * R.row_blocks;
        b = (int)fdiv((unsigned)bh, R.by_heads), h = bh - b * A.kv_heads;
        return u < R.units;
    };
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();

    if (warp == kRowWarps) {
        // ------------------------------------------------------------------------------------------------ the requests
        // Lane k serves ring k, so that a pass over the rings costs as much as one of them.
        int rb, b = 0, h = 0, len = 0, pc = 0, c1 = 0;
        if (lane < rings && unit_of(lane, rb, b, h)) {
            len = states_of(A, b);
            // this ring's chunks: all, or its run of the cluster's
            c1 = (len + P::CHUNK - 1) / P::CHUNK;
            if (!R.whole) {
                const int w = rank * rings + lane, each = (int)fdiv((unsigned)c1, R.by_workers), more = c1 - each * (R.splits * rings);
                pc = w * each + min(w, more), c1 = pc + each + (w < more);
            }
        }
        bool more = lane < rings, ok = true;
        int slot = 0, use = 0;
        // A mask is read eight chunks at a time, of all rings at once: lane 8 k + i holds the truth values of chunk wb + i of ring k. (32 x 17
        // queries over 2560 states, 32 heads of 48, L2 flushed: all states there 125 -> 115 us, every 256th 64 -> 41, none 49 -> 29.)
        int wb = pc - 8;
        u32 win = 0;
        u32 s = lane * stages, dst = sbase + s * P::STAGE, full = bars + 16 * s;      // of this lane's ring and the pass's stage
        while (ok && __any_sync(0xffffffffu, more)) {
            u32 bits = 0;
            if (!A.mask) {
                const int n = len - pc * P::CHUNK;
                bits = n >= P::CHUNK ? kAll : n <= 0 ? 0u : (1u << n) - 1u;
                if (pc >= c1) bits = 0;
            } else {
                // the next chunk that holds a state: in the window, or in the next ones
                u32 mine;
                for (;;) {
                    const u32 any = __ballot_sync(0xffffffffu, win != 0);
                    mine = lane < RINGS ? any >> (8 * lane) & (0xffu << (pc - wb)) & 0xffu : 0u;
                    const bool need = more && mine == 0 && wb + 8 < c1;
                    const u32 needs = __ballot_sync(0xffffffffu, need);
                    if (!needs) break;
                    if (need) wb += 8, pc = wb;
                    unsigned char x[RINGS][8];
#pragma unroll
                    for (int k = 0; k < RINGS; ++k) {
                        const int at = __shfl_sync(0xffffffffu, wb, k), end = __shfl_sync(0xffffffffu, c1, k), n = __shfl_sync(0xffffffffu, len, k);
                        const unsigned char* row = A.mask + __shfl_sync(0xffffffffu, b, k) * A.mask_sb;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int j = (at + i) * P::CHUNK + lane;
                            x[k][i] = needs >> k & 1 && lane < P::CHUNK && at + i < end && j < n ? row[j] : 0;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < RINGS; ++k)
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const u32 y = __ballot_sync(0xffffffffu, x[k][i] != 0);
                            if (needs >> k & 1 && lane == 8 * k + i) win = y;
                        }
                }
                const int i = mine ? __ffs(mine) - 1 : 0;
                bits = __shfl_sync(0xffffffffu, win, (8 * lane + i) & 31);
                if (mine) pc = wb + i;
                else pc = c1, bits = 0;
            }
            if (more) {
                if (use) ok = mbar_wait_ready(full + 8, (use - 1) & 1, abort_flag, &g_tcq_cross_error);
                if (ok) {
                    meta[s] = make_int2(bits ? pc : -1, (int)bits);
                    if (!bits) {
                        mbar_arrive(full);
                        more = false;
                    } else {
                        mbar_expect_tx(full, P::STAGE);
#pragma unroll
                        for (int a = 0; a < P::ATOMS; ++a) tma_load_4d(dst + a * (P::CHUNK * 128), &kmap, full, 64 * a, pc * P::CHUNK, h, b * A.kb);
#pragma unroll
                        for (int a = 0; a < P::ATOMS; ++a) tma_load_4d(dst + P::HALF + a * (P::CHUNK * 128), &vmap, full, 64 * a, pc * P::CHUNK, h, b * A.vb);
                        ++pc;
                    }
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            ++s, dst += P::STAGE, full += 16;
            if (++slot == stages) slot = 0, ++use, s -= stages, dst -= stages * P::STAGE, full -= 16 * stages;
        }
        if (*abort_flag && lane < rings) {                         // copies on their way land before their stages are left
            volatile int never = 0;
            for (int i = 0; i < stages; ++i) {
                const int uses = use + (i < slot);                 // at most: a barrier that saw fewer is waited for in vain, within the limit
                if (uses) mbar_wait_suspended(bars + 16 * (lane * stages + i), (uses - 1) & 1, &never, &g_tcq_cross_error, kWaitNs / 100);
            }
        }
        __syncwarp();
        if (R.whole || rings * R.splits == 1) return;
        __syncthreads();
        if (R.splits > 1) cluster_barrier(), cluster_barrier();
        return;
    }

    // ------------------------------------------------------------------------------------------------ this warp's rows: 16 j + g, + 8
    int rb, b, h;
    const bool there = unit_of(kg, rb, b, h);
    const int w0 = P::ROWS * wm, r0 = rb * R.block_rows, r1 = there ? min(A.rows, r0 + R.block_rows) : 0;
    const bool live = r0 + w0 < r1;                                // a warp without a row only keeps the barriers going
    u32 q[MT][KS][4];
    {
        const u32 flip = query_flip(A), keep = query_keep(A);
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = r0 + w0 + 16 * j + 8 * e + g;
                const u16* qr = A.q + row_at(A, b, h, min(r, A.rows - 1), A.q_sb, A.q_st);
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int d = 16 * k + 8 * x + 2 * t;
                        q[j][k][2 * x + e] = d < A.D && r < r1 ? *reinterpret_cast<const u32*>(qr + d) : 0u;
                    }
            }
        if (flip || !keep) {
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[j][k][e] = q[j][k][e] & keep ^ flip;
        }
    }
    const float c = score_scale(A);
    float o[MT][NT][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        m[j][0] = m[j][1] = -INFINITY, l[j][0] = l[j][1] = 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
    }

    // One chunk: the scores of its states, weights, O += P V. Matrices of 8 x 8 are read from the swizzled tiles: 16-byte piece p of row r
    // lies at p ^ (r & 7). Products that add to the same registers are issued as far apart as they can be.
    const int row8 = lane & 7, row16 = lane & 15;
    auto chunk = [&](auto masked_c, u32 bits, u32 kt, u32 vt) {
        constexpr bool MASKED = decltype(masked_c)::value;
        float s[MT][NK][4];
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int n = 0; n < NK; ++n) s[j][n][0] = s[j][n][1] = s[j][n][2] = s[j][n][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
            const int p = 2 * k + (lane >> 3);                     // pieces of 8 elements: two of step k, two of step k + 1
            u32 f[NK][4];
#pragma unroll
            for (int n = 0; n < NK; ++n) ldsm4(kt + (p >> 3) * (P::CHUNK * 128) + (8 * n + row8) * 128 + (((p & 7) ^ row8) << 4), f[n]);
#pragma unroll
            for (int x = 0; x < 2 && k + x < KS; ++x)
#pragma unroll
                for (int n = 0; n < NK; ++n)
#pragma unroll
                    for (int j = 0; j < MT; ++j)
                        mma16816<DT>(s[j][n], q[j][k + x][0], q[j][k + x][1], q[j][k + x][2], q[j][k + x][3], f[n][2 * x], f[n][2 * x + 1]);
        }
        if (MASKED) {
            const u32 w = bits >> (2 * t);
#pragma unroll
            for (int n = 0; n < NK; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (!(w >> (8 * n + e) & 1)) {
#pragma unroll
                        for (int j = 0; j < MT; ++j) s[j][n][e] = s[j][n][2 + e] = -INFINITY;
                    }
        }
        float top[MT][2];
        bool above = false;
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[j][e] = fmaxf(s[j][0][2 * e], s[j][0][2 * e + 1]);
#pragma unroll
                for (int n = 1; n < NK; ++n) top[j][e] = max3(top[j][e], s[j][n][2 * e], s[j][n][2 * e + 1]);
                top[j][e] *= c;
                above = above || top[j][e] > m[j][e] + kSlack;
            }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = top[j][e];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    const bool move = x > m[j][e] + kSlack;
                    f[e] = move ? ex2(m[j][e] - x) : 1.f;
                    if (move) m[j][e] = x;
                    l[j][e] *= f[e];
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) o[j][i][0] *= f[0], o[j][i][1] *= f[0], o[j][i][2] *= f[1], o[j][i][3] *= f[1];
            }
        }
        const u64 c2 = pair(c, c);
        u32 w[MT][NK][2];                                          // weights of rows g and g + 8
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float base = kRef - (m[j][e] == -INFINITY ? 0.f : m[j][e]);
                const u64 b2 = pair(base, base);
                u64 sum = 0;
                float lo, hi;
#pragma unroll
                for (int n = 0; n < NK; ++n) {
                    unpair(fma2(pair(s[j][n][2 * e], s[j][n][2 * e + 1]), c2, b2), lo, hi);
                    lo = ex2(lo), hi = ex2(hi);
                    sum = add2(sum, pair(lo, hi));
                    w[j][n][e] = weights2<DT>(lo, hi);
                }
                unpair(sum, lo, hi);
                l[j][e] += lo + hi;
            }
#pragma unroll
        for (int k = 0; k < NK / 2; ++k) {
            // what lies where no state is may be anything, NaN too: this lane's keys 16 k + 2 t, + 1 and 8 further
            u32 z0 = 0xffffffffu, z1 = 0xffffffffu;
            if (MASKED) {
                const u32 x = bits >> (16 * k + 2 * t);
                z0 = (x & 1 ? 0xffffu : 0u) | (x & 2 ? 0xffff0000u : 0u);
                z1 = (x & 256 ? 0xffffu : 0u) | (x & 512 ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int i = 0; i < NT; i += 2) {
                u32 f[4];
                const int p = i + (lane >> 4);
                ldsm4t(vt + (p >> 3) * (P::CHUNK * 128) + (16 * k + row16) * 128 + (((p & 7) ^ row8) << 4), f);
                if (MASKED) f[0] &= z0, f[1] &= z1, f[2] &= z0, f[3] &= z1;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int j = 0; j < MT; ++j)
                        mma16816<DT>(o[j][i + x], w[j][2 * k][0], w[j][2 * k][1], w[j][2 * k + 1][0], w[j][2 * k + 1][1], f[2 * x], f[2 * x + 1]);
            }
        }
    };
    int slot = kg * stages;
    u32 phase = 0;
    for (;;) {
        if (!mbar_wait_ready(bars + 16 * slot, phase, abort_flag, &g_tcq_cross_error)) break;
        const int2 what = meta[slot];
        if (what.x < 0) break;
        const u32 kt = sbase + slot * P::STAGE;
        if (live) {
            if ((u32)what.y == kAll) chunk(std::false_type(), kAll, kt, kt + P::HALF);
            else chunk(std::true_type(), (u32)what.y, kt, kt + P::HALF);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + 16 * slot + 8);
        if (++slot == (kg + 1) * stages) slot = kg * stages, phase ^= 1;
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 1);
            l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 2);
        }
    const i64 out_st = (i64)A.heads * A.D, out_sb = (i64)A.T * out_st;
    if (R.whole || rings * R.splits == 1) {
        // (sixteen bytes a lane, turned among the four of a row by shuffles, took ten times as long)
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = r0 + w0 + 16 * j + 8 * e + g;
                const float f = l[j][e] != 0.f ? 1.f / l[j][e] : 0.f;
                u32* dst = reinterpret_cast<u32*>(A.out + row_at(A, b, h, min(r, A.rows - 1), out_sb, out_st));
                if (r < r1)
#pragma unroll
                    for (int i = 0; i < NT; ++i)
                        if (8 * i < A.D) dst[4 * i + t] = weights2<DT>(o[j][i][2 * e] * f, o[j][i][2 * e + 1] * f);
            }
        bool past = false;                                         // behind the stores, which do not wait for it
#pragma unroll
        for (int j = 0; j < MT; ++j) past = past || past_range(m[j][0]) || past_range(m[j][1]);
        if (past) atomicOr(&g_tcq_cross_error, 2);
        return;
    }
    // ---- parts to shared memory (every chunk has arrived), then added: four elements of a row a thread
    __syncthreads();
    float* const parts = reinterpret_cast<float*>(smem_rows);
    {
        float* part = parts + (size_t)(kg * WM + wm) * P::ROWS * P::PITCH;
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float* row = part + (16 * j + 8 * e + g) * P::PITCH;
#pragma unroll
                for (int i = 0; i < NT; ++i) *reinterpret_cast<float2*>(row + 8 * i + 2 * t) = make_float2(o[j][i][2 * e], o[j][i][2 * e + 1]);
                if (t == 0) *reinterpret_cast<float2*>(row + DP) = make_float2(m[j][e], l[j][e]);
            }
    }
    const int rows = r1 - r0;
    bool past = false;
    auto store = [&](int row, int d, const float4& y, float top, float sum) {
        const float f = sum != 0.f ? 1.f / sum : 0.f;
        if (d < A.D)
            *reinterpret_cast<uint2*>(A.out + row_at(A, b, h, r0 + row, out_sb, out_st) + d) = make_uint2(weights2<DT>(y.x * f, y.y * f), weights2<DT>(y.z * f, y.w * f));
        past = past || past_range(top);
    };
    asm volatile("barrier.cta.sync 1, %0;" ::"n"(32 * kRowWarps) : "memory");
    for (int i = tid; i < rows * (DP / 4); i += 32 * kRowWarps) {
        const int row = i / (DP / 4), d = 4 * (i - row * (DP / 4));
        const float* p = parts + row * P::PITCH;
        float2 ml[RINGS];
        float4 v[RINGS], y = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < RINGS; ++k) {
            ml[k] = make_float2(-INFINITY, 0.f), v[k] = y;
            if (k < rings) {
                ml[k] = *reinterpret_cast<const float2*>(p + k * WM * P::ROWS * P::PITCH + DP);
                v[k] = *reinterpret_cast<const float4*>(p + k * WM * P::ROWS * P::PITCH + d);
            }
            top = fmaxf(top, ml[k].x);
        }
#pragma unroll
        for (int k = 0; k < RINGS; ++k) {
            const float f = part_factor(ml[k], top);
            sum = __fmaf_rn(ml[k].y, f, sum);
            y.x = __fmaf_rn(v[k].x, f, y.x), y.y = __fmaf_rn(v[k].y, f, y.y), y.z = __fmaf_rn(v[k].z, f, y.z), y.w = __fmaf_rn(v[k].w, f, y.w);
        }
        if (R.splits == 1) {
            store(row, d, y, top, sum);
        } else {
            *reinterpret_cast<float4*>(parts + row * P::PITCH + d) = y;             // read by no other thread before
            if (d == 0) *reinterpret_cast<float2*>(smem_rows + P::PARTS + 8 * row) = make_float2(top, sum);
        }
    }
    if (R.splits == 1) {
        if (past) atomicOr(&g_tcq_cross_error, 2);
        return;
    }
    cluster_barrier();
    for (int i = rank * (32 * kRowWarps) + tid; i < rows * (DP / 4); i += R.splits * (32 * kRowWarps)) {
        const int row = i / (DP / 4), d = 4 * (i - row * (DP / 4));
        // four parts at a time, all of their loads under way at once
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, sum = 0.f;
        for (int k0 = 0; k0 < R.splits; k0 += 4) {
            float2 ml[4];
            float4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                ml[k] = make_float2(-INFINITY, 0.f), v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k0 + k < R.splits) {
                    const u32 p = peer_addr(sbase, k0 + k);
                    ml[k] = peer_ld2(p + P::PARTS + 8 * row);
                    v[k] = peer_ld4(p + (row * P::PITCH + d) * 4);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float both = fmaxf(top, ml[k].x), old = both == -INFINITY ? 1.f : ex2(top - both), f = part_factor(ml[k], both);
                top = both;
                sum = __fmaf_rn(ml[k].y, f, sum * old);
                y.x = __fmaf_rn(v[k].x, f, y.x * old), y.y = __fmaf_rn(v[k].y, f, y.y * old);
                y.z = __fmaf_rn(v[k].z, f, y.z * old), y.w = __fmaf_rn(v[k].w, f, y.w * old);
            }
        }
        store(row, d, y, top, sum);
    }
    if (past) atomicOr(&g_tcq_cross_error, 2);
    __syncwarp();
    cluster_barrier();                                             // a part may be read until here
}

// ------------------------------------------------------------------------------------------------ tiles of 128 rows
// Tensor-core products (tcgen05) on tiles of 128 query rows and 128 states, for many rows over many states. A CTA has two groups
// of softmax warps, 128 threads each, a row to a thread. ROWS: the groups take 128 rows each of one unit (up to 256 rows of one key
// head) and every tile of states serves both. Otherwise (up to 128 rows) both groups take the same rows and every other tile each, and
// their parts are added at the end. Roles:
//   softmax   scores from TMEM into registers, weights back over the scores (16 bits, 64 of the 128 columns), half a tile at a time;
//   product   one warp, an elected lane of which issues S = Q K^T (Q, K in shared memory) and O += P V (P in TMEM, V as it lies in
//             memory: the states along the contraction, MN-major);
//   load      one warp: which tiles hold a state, their truth values as bits, K and V into a ring of tiles (TMA);
//   clean     one warp, only where lens or a mask may leave states out: rows of V without a state become zero before a product reads
//             them (a weight of zero times NaN is NaN). Keys need no such care: their scores are replaced.
// The groups alternate: while one's weights are formed, the other's products run. A group's S of a tile is issued after its O
// of the tile before, and a commit covers every product issued before it: scores that have arrived mean that O is complete
// up to the tile before. The reference m of a row moves only when a score passes it by kSlack; O (in TMEM) is then
// rescaled by its own row's thread.
//
// Bound by the products' shared-memory operands (a tile for both groups at head width 128 takes 3,100 clocks, with the exponentials left out 2,900,
// where its products alone should take 2,048) and, below that width, by the chain scores - maximum - weights (a warp alone gets an
// exponential in 11 clocks of the unit's 8; 2,830 clocks a tile at width 64): 2 x 4096 x 4096, 32 heads of 128 over 8 (F16) 449 to 455 us,
// 1,208 to 1,224 TFLOP/s; heads of 64 374 us. Measured on the way, the first of these: queries requested one by one 544 us, the waits' loop
// entered for complete barriers 468. No faster: scores in two halves 521, two threads to a row 464 (against 465), a product warp for each group
// 459 (454), an eighth of the exponentials by polynomial 466 (454), the groups taking turns at the exponentials 474 (454).
constexpr int kTile = 128;
template <int DP, bool ROWS>
struct Tiles {
    static constexpr int ATOMS = (DP + 63) / 64;                       // 64-element columns of a tile
    static constexpr int TB = ATOMS * kTile * 128;                     // bytes of a tile: a group's queries, keys, values
    static constexpr int QN = ROWS ? 2 : 1;
    static constexpr int FIT = (226 * 1024 - QN * TB) / TB, RING = FIT < 8 ? FIT : 8;      // tiles of keys and values on their way
    // Eight softmax warps; product, load and clean warps and one that only makes the warpgroup whole. The CTA is launched with 168 registers
    // a thread (384 x 168 = 64,512); the softmax warps take 208 and the others keep 88: 256 x 208 + 128 x 88 = 64,512.
    static constexpr int THREADS = 384, LAUNCH_REGS = 168;
    static constexpr int Q0 = 0, RING0 = QN * TB, BAR0 = RING0 + RING * TB;
    static constexpr int META = 8;                                     // tiles whose truth values are kept
    static constexpr int META0 = BAR0 + 304, ML0 = META0 + META * 32;  // m, l of every row
    static constexpr int BYTES = ML0 + 2 * kTile * 8;
    // TMEM columns: scores (128 each), outputs. Up to head width 64 the weights have columns of their own, so that the next tile's scores
    // may be formed while the weights of this one are; else they lie over the scores.
    static constexpr bool EARLY = DP <= 64;
    static constexpr u32 COLS = 512, S0 = 0, P0 = EARLY ? 256 : 0, PG = EARLY ? 64 : 128, O0 = EARLY ? 384 : 256, OG = EARLY ? 64 : 128;
    static constexpr int PARTS = 2 * kTile * DP * 4;
    static_assert(RING >= 5, "two tiles in use, the next keys on their way");
    static_assert(PARTS <= BAR0 && BYTES <= 227 * 1024, "the parts overlay the tiles");
};
// What is kept of a tile: its number (below 0: the end), whether all its states are there, its truth values.
struct TileMeta {
    int at, whole, pad[2];
    u32 bits[4];
};
// Barriers, 8 bytes each from BAR0: ring slot i full and empty, values of tile t cleaned (t mod META), of group g scores, weights
// (two halves), scores read and outputs (EARLY), queries, the end.
enum { TBAR_FULL = 0, TBAR_EMPTY = 8, TBAR_CLEAN = 16, TBAR_S = 24, TBAR_P = 26, TBAR_READ = 30, TBAR_O = 32, TBAR_Q = 34, TBAR_END = 35, TBAR_COUNT = 36 };


// Boxes of a whole tile's states, and of half a tile's (only where a mask may leave blocks out between two that are wanted: a tile in two
// boxes costs 7 % of the whole call, 2 x 4096 x 4096, heads of 128, 456 -> 488 us).
struct TileMaps {
    CUtensorMap k, v, k_half, v_half;
};
struct TilesPlan {
    int row_tiles, tile_rows, splits;
    FastDiv by_tiles, by_heads, by_splits;
};

template <int DT, int DP, bool ROWS>
__global__ void __launch_bounds__(Tiles<DP, ROWS>::THREADS, 1)
k_cross_tiles(const CrossArgs A, const __grid_constant__ TileMaps maps, const TilesPlan R) {
    typedef Tiles<DP, ROWS> P;
    constexpr int KS = DP / 16;
    constexpr u32 IDESC = DT == TCQ_DT_BF16 ? kIdescBf16 : 0u;
    extern __shared__ __align__(1024) char smem_tiles[];
    char* const smem = smem_tiles;
    const u32 sbase = smem_u32(smem), bars = sbase + P::BAR0;
    u32* tmem_slot = reinterpret_cast<u32*>(smem + P::BAR0 + 8 * TBAR_COUNT);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + P::META0) + 2;      // in the first entry's padding
    TileMeta* meta = reinterpret_cast<TileMeta*>(smem + P::META0);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    constexpr int W_MMA = 8, W_LOAD = 9, W_CLEAN = 10;
    auto bar = [&](int i) -> u32 { return bars + 8 * i; };
    auto wait = [&](int i, u32 parity) -> bool { return mbar_wait_ready(bar(i), parity & 1, abort_flag, &g_tcq_cross_error); };
    if (tid == 0) {
        for (int i = 0; i < P::RING; ++i) {
            mbar_init(bar(TBAR_FULL + i), 1);
            mbar_init(bar(TBAR_EMPTY + i), 1);
        }
        for (int i = 0; i < P::META; ++i) mbar_init(bar(TBAR_CLEAN + i), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(TBAR_S + i), 1);
            mbar_init(bar(TBAR_READ + i), 4);
            mbar_init(bar(TBAR_O + i), 1);
            mbar_init(bar(TBAR_P + 2 * i), 4);                // per softmax warp; group and half at 2 g + half
            mbar_init(bar(TBAR_P + 2 * i + 1), 4);
        }
        mbar_init(bar(TBAR_Q), 256);
        mbar_init(bar(TBAR_END), 1);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(P::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const u32 tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    // ---- the unit: rows r0 .. r1 - 1 of key head h of sequence b, and this CTA's half tiles [k0, k1) of its states
    const int splits = R.splits, unit = (int)fdiv(blockIdx.x, R.by_splits), sp = (int)blockIdx.x - unit * splits;
    const int bh = (int)fdiv((unsigned)unit, R.by_tiles), b = (int)fdiv((unsigned)bh, R.by_heads), h = bh - b * A.kv_heads;
    const int r0 = (unit - bh * R.row_tiles) * R.tile_rows, r1 = min(A.rows, r0 + R.tile_rows);
    const int len = states_of(A, b), tiles = (len + kTile - 1) / kTile;
    const int each = (int)fdiv((unsigned)tiles, R.by_splits), more = tiles - each * splits, first = sp * each + min(sp, more);
    const int k0 = 2 * first, k1 = min(2 * (first + each + (sp < more)), (len + kTile / 2 - 1) / (kTile / 2));
    const bool parts = splits > 1 || !ROWS;                   // rows have more than one part
    const bool ragged = A.lens || A.mask;

    if (warp < W_MMA) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < W_MMA) {
        // ------------------------------------------------------------------------------------------------ softmax
        const int g = warp >> 2, gl = tid & 127, row = ROWS ? g * kTile + gl : gl;
        const bool idle = r0 + (row & ~31) >= r1;             // a warp without a row only keeps the barriers going
        const float c = score_scale(A);
        constexpr int SEG = DP <= 32 ? 4 : DP <= 64 ? 8 : 16, RPP = 32 / SEG;      // lanes to a row of 16-byte pieces, rows a pass
        if (k1 > k0) {
            // queries to shared memory, all of a thread's requested at once
            constexpr int WROWS = ROWS ? 32 : 16, NP = WROWS / RPP;
            const int sl = lane % SEG, first = warp * WROWS;
            const u32 flip = query_flip(A), keep = query_keep(A);
            uint4 w[NP];
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const int rr = r0 + first + n * RPP + lane / SEG;
                w[n] = make_uint4(0, 0, 0, 0);
                if (rr < r1 && 8 * sl < A.D) w[n] = *reinterpret_cast<const uint4*>(A.q + row_at(A, b, h, rr, A.q_sb, A.q_st) + 8 * sl);
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const int q = first + n * RPP + lane / SEG, qg = q >> 7, qr = q & 127;
                w[n].x = w[n].x & keep ^ flip, w[n].y = w[n].y & keep ^ flip, w[n].z = w[n].z & keep ^ flip, w[n].w = w[n].w & keep ^ flip;
                if (8 * sl < DP)
                    *reinterpret_cast<uint4*>(smem + P::Q0 + qg * P::TB + (sl >> 3) * (kTile * 128) + qr * 128 + (((sl & 7) ^ (qr & 7)) << 4)) = w[n];
            }
            async_proxy_fence();
        }
        mbar_arrive(bar(TBAR_Q));
        const u32 lanes = (u32)((warp & 3) * 32) << 16, ts = tmem + lanes + P::S0 + g * kTile, tp = tmem + lanes + P::P0 + g * P::PG,
                  to = tmem + lanes + P::O0 + g * P::OG;
        float m = -INFINITY, l = 0.f;
        // One tile: 128 scores of this thread's row, their largest, weights over them. Nothing of the scores is read after the first
        // store; the product of a half is issued when its four warps have handed it over.
        auto tile = [&](auto masked_c, int i, const u32 (&bits)[4]) -> bool {
            constexpr bool MASKED = decltype(masked_c)::value;
            u32 v[4][32];
            float raw[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            tmem_ld32(ts, v[0]);
            tmem_ld32(ts + 32, v[1]);
            tmem_ld_wait(v[0]);
            tmem_ld_wait(v[1]);
            tmem_ld32(ts + 64, v[2]);
            tmem_ld32(ts + 96, v[3]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (half) {
                    tmem_ld_wait(v[2]);
                    tmem_ld_wait(v[3]);
                    if (P::EARLY) {
                        tc_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar(TBAR_READ + g));
                    }
                }
                if (MASKED) {
#pragma unroll
                    for (int j = 64 * half; j < 64 * half + 64; ++j)
                        if (!(bits[j >> 5] >> (j & 31) & 1)) v[j >> 5][j & 31] = 0xff800000u;
                }
#pragma unroll
                for (int j = 64 * half; j < 64 * half + 64; j += 2)
                    raw[(j >> 1) & 3] = max3(raw[(j >> 1) & 3], __uint_as_float(v[j >> 5][j & 31]), __uint_as_float(v[j >> 5][(j & 31) + 1]));
            }
            if (P::EARLY && i > 0) {                          // the outputs up to the tile before are complete, its weights used
                if (!wait(TBAR_O + g, i - 1)) return false;
                tc_after();
            }
            float top = fmaxf(fmaxf(raw[0], raw[1]), fmaxf(raw[2], raw[3]));
            top *= c;
            if (__any_sync(0xffffffffu, top > m + kSlack)) {
                const bool move = top > m + kSlack;
                const float f = move ? ex2(m - top) : 1.f;
                if (move) m = top;
                l *= f;
                if (i > 0) {
#pragma unroll 1
                    for (int d = 0; d < DP; d += 16) {
                        u32 o[2][8];
                        tmem_ld8(to + d, o[0]);
                        tmem_ld8(to + d + 8, o[1]);
                        tmem_ld_wait(o[0]);
                        tmem_ld_wait(o[1]);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            o[0][j] = __float_as_uint(__uint_as_float(o[0][j]) * f), o[1][j] = __float_as_uint(__uint_as_float(o[1][j]) * f);
                        tmem_st8(to + d, o[0]);
                        tmem_st8(to + d + 8, o[1]);
                    }
                }
            }
            const float base = kRef - (m == -INFINITY ? 0.f : m);
            const u64 c2 = pair(c, c), a2 = pair(base, base);
            u64 sum[2] = {0, 0};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                u32 w[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const u64 x = fma2(pair(__uint_as_float(v[q][2 * j]), __uint_as_float(v[q][2 * j + 1])), c2, a2);
                    float lo, hi;
                    unpair(x, lo, hi);
                    lo = ex2(lo), hi = ex2(hi);
                    sum[j & 1] = add2(sum[j & 1], pair(lo, hi));
                    w[j] = weights2<DT>(lo, hi);
                }
                tmem_st16(tp + 16 * q, w);
                if (q & 1) {
                    tmem_st_wait();
                    tc_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(TBAR_P + 2 * g + (q >> 1)));
                }
            }
            float lo, hi;
            unpair(add2(sum[0], sum[1]), lo, hi);
            l += lo + hi;
            return true;
        };
        bool ok = true;
        for (int i = 0; k1 > k0; ++i) {
            ok = wait(TBAR_S + g, i);
            tc_after();
            if (!ok) break;
            const TileMeta& t = meta[(ROWS ? i : 2 * i + g) & (P::META - 1)];
            const int4 head = *reinterpret_cast<const int4*>(&t);
            if (head.x < 0) break;
            if (idle) {
                // the next scores may come before the other warps have handed this tile's weights over: not before its outputs
                if (P::EARLY && i > 0) ok = wait(TBAR_O + g, i - 1);
                if (!ok) break;
                if (lane == 0) {
                    if (P::EARLY) mbar_arrive(bar(TBAR_READ + g));
                    mbar_arrive(bar(TBAR_P + 2 * g)), mbar_arrive(bar(TBAR_P + 2 * g + 1));
                }
                continue;
            }
            u32 bits[4] = {};
            if (head.y) {
                ok = tile(std::false_type(), i, bits);
            } else {
                const uint4 w = *reinterpret_cast<const uint4*>(t.bits);
                bits[0] = w.x, bits[1] = w.y, bits[2] = w.z, bits[3] = w.w;
                ok = tile(std::true_type(), i, bits);
            }
            if (!ok) break;
        }
        // every product has ended: the rows' outputs, or their parts, over the tiles, 16-byte pieces permuted within a row
        const bool got = ok && l != 0.f;
        const float f = parts ? 1.f : got ? 1.f / l : 0.f;
        if (parts) asm volatile("barrier.cta.sync 15, 256;" ::: "memory");
        constexpr int XP = (DP / 4) % 8 == 0 ? 7 : 3, XO = (DP / 8) % 8 == 0 ? 7 : (DP / 8) % 4 == 0 ? 3 : 1;
        if (!idle) {
#pragma unroll
            for (int d0 = 0; d0 < DP; d0 += 32) {
                u32 o[32] = {};
                if (ok && k1 > k0) {
                    if (d0 + 32 <= DP) tmem_ld32(to + d0, o);
                    else tmem_ld16(to + d0, o);
                    tmem_ld_wait(o);
                }
#pragma unroll
                for (int d = d0; d < d0 + 32 && d < DP; d += 8) {
                    float y[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = got ? __uint_as_float(o[d - d0 + j]) * f : 0.f;
                    if (parts) {
                        float4* part = reinterpret_cast<float4*>(smem) + (g * kTile + gl) * (DP / 4);
                        part[(d / 4) ^ (gl & XP)] = make_float4(y[0], y[1], y[2], y[3]);
                        part[(d / 4 + 1) ^ (gl & XP)] = make_float4(y[4], y[5], y[6], y[7]);
                    } else {
                        reinterpret_cast<uint4*>(smem + P::Q0 + g * P::TB)[gl * (DP / 8) + ((d / 8) ^ (gl & XO))] =
                            make_uint4(weights2<DT>(y[0], y[1]), weights2<DT>(y[2], y[3]), weights2<DT>(y[4], y[5]), weights2<DT>(y[6], y[7]));
                    }
                }
            }
        }
        if (parts) {
            reinterpret_cast<float2*>(smem + P::ML0)[g * kTile + gl] = make_float2(ok && !idle ? m : -INFINITY, ok && !idle ? l : 0.f);
        } else if (!idle) {
            __syncwarp();
            const int sl = lane % SEG;
#pragma unroll 4
            for (int n = 0; n < 32; n += RPP) {
                const int rr = (gl & ~31) + n + lane / SEG, rg = r0 + (row & ~31) + n + lane / SEG;
                if (rg < r1 && 8 * sl < A.D) {
                    u16* dst = A.out + row_at(A, b, h, rg, (i64)A.T * A.heads * A.D, (i64)A.heads * A.D);
                    reinterpret_cast<uint4*>(dst)[sl] = reinterpret_cast<const uint4*>(smem + P::Q0 + g * P::TB)[rr * (DP / 8) + (sl ^ (rr & XO))];
                }
            }
        }
        if (past_range(m)) atomicOr(&g_tcq_cross_error, 2);
    } else if (k1 > k0 && warp == W_LOAD) {
        // ------------------------------------------------------------------------------------------------ load
        // A tile is made of the next two blocks of 64 states that hold one, so that what a mask leaves out in such blocks (an image) costs
        // nothing. Item 2 t of the ring is the keys of tile t, item 2 t + 1 its values.
        constexpr int H = kTile / 2;
        const unsigned char* mrow = A.mask ? A.mask + b * A.mask_sb : nullptr;
        unsigned char mb[2] = {};
        int i = k0;
        auto look = [&]() {                                   // the truth values of block i
            if (mrow && i < k1)
#pragma unroll
                for (int j = 0; j < 2; ++j) mb[j] = i * H + 32 * j + lane < len ? mrow[i * H + 32 * j + lane] : 0;
        };
        auto next = [&](u32& w0, u32& w1) -> int {            // the next block with a state, its truth values; below 0: none
            w0 = w1 = 0;
            while (i < k1) {
                const int n = len - i * H;
                w0 = mrow ? __ballot_sync(0xffffffffu, mb[0] != 0) : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
                w1 = mrow ? __ballot_sync(0xffffffffu, mb[1] != 0) : n >= 64 ? 0xffffffffu : n > 32 ? (1u << (n - 32)) - 1u : 0u;
                ++i;
                look();
                if (w0 | w1) return i - 1;
            }
            return -1;
        };
        look();
        bool ok = true;
        int t = 0;
        auto slot_free = [&](int item) { return item < P::RING || wait(TBAR_EMPTY + item % P::RING, item / P::RING - 1); };
        while (ok) {
            u32 w[4];
            const int b0 = next(w[0], w[1]);
            if (b0 < 0) break;
            const int b1 = next(w[2], w[3]);
            // Neighbours, or the last block alone, are one box: what it has too much is not there, rows past the last state arrive as zeros.
            const bool one = b1 < 0 || b1 == b0 + 1;
            ok = slot_free(2 * t);
            if (ok && lane == 0) {
                TileMeta& e = meta[t & (P::META - 1)];
                e.at = b0, e.whole = (w[0] & w[1] & w[2] & w[3]) == 0xffffffffu;
                e.bits[0] = w[0], e.bits[1] = w[1], e.bits[2] = w[2], e.bits[3] = w[3];
            }
            for (int vals = 0; vals < 2 && ok; ++vals) {
                const int item = 2 * t + vals, s = item % P::RING;
                if (vals) ok = slot_free(item);
                if (ok && lane == 0) {
                    const u32 dst = sbase + P::RING0 + s * P::TB;
                    const int sequence = b * (vals ? A.vb : A.kb);
                    mbar_expect_tx(bar(TBAR_FULL + s), P::TB);
#pragma unroll
                    for (int a = 0; a < P::ATOMS; ++a) {
                        const u32 to = dst + a * (kTile * 128);
                        if (one) {
                            tma_load_4d(to, vals ? &maps.v : &maps.k, bar(TBAR_FULL + s), 64 * a, b0 * H, h, sequence);
                        } else {
                            tma_load_4d(to, vals ? &maps.v_half : &maps.k_half, bar(TBAR_FULL + s), 64 * a, b0 * H, h, sequence);
                            tma_load_4d(to + H * 128, vals ? &maps.v_half : &maps.k_half, bar(TBAR_FULL + s), 64 * a, b1 * H, h, sequence);
                        }
                    }
                }
                __syncwarp();
            }
            if (ok) ++t;
        }
        // the end, for the product and clean warps: in place of the next keys (and, where the groups take turns, of those behind them)
        for (int e = 0; e < (ROWS ? 1 : 2) && ok; ++e) {
            ok = slot_free(2 * (t + e)) && slot_free(2 * (t + e) + 1);
            if (ok && lane == 0) {
                meta[(t + e) & (P::META - 1)].at = -1;
                mbar_arrive(bar(TBAR_FULL + 2 * (t + e) % P::RING));
                mbar_arrive(bar(TBAR_FULL + (2 * (t + e) + 1) % P::RING));
            }
            __syncwarp();
        }
        if (*abort_flag) {                                    // copies on their way land before the CTA ends
            volatile int never = 0;
            for (int item = max(0, 2 * t - P::RING); item < 2 * t; ++item)
                mbar_wait_suspended(bar(TBAR_FULL + item % P::RING), (item / P::RING) & 1, &never, &g_tcq_cross_error, kWaitNs / 20);
        }
    } else if (k1 > k0 && warp == W_CLEAN && ragged) {
        // ------------------------------------------------------------------------------------------------ clean
        for (int t = 0;; ++t) {
            const int item = 2 * t + 1, s = item % P::RING;
            if (!wait(TBAR_FULL + s, item / P::RING)) break;
            const TileMeta& e = meta[t & (P::META - 1)];
            if (e.at < 0) break;
            if (!e.whole) {
                char* v = smem + P::RING0 + s * P::TB;
                for (int j = 0; j < kTile; j += 4) {
                    const int key = j + (lane >> 3);             // eight lanes to a row of 128 bytes
                    if (!(e.bits[key >> 5] >> (key & 31) & 1))
#pragma unroll
                        for (int a = 0; a < P::ATOMS; ++a) *reinterpret_cast<uint4*>(v + a * (kTile * 128) + key * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                async_proxy_fence();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(TBAR_CLEAN + (t & (P::META - 1))));
        }
    } else if (k1 > k0 && warp == W_MMA) {
        // ------------------------------------------------------------------------------------------------ product
        const u64 qd = sw128_desc(sbase + P::Q0), kd = sw128_desc(sbase + P::RING0), vd = sw128_desc_mn(sbase + P::RING0, kTile * 128);
        constexpr u32 atom = kTile * 128 / 16, tb = P::TB >> 4;
        bool ended[2] = {false, false};
        // S of group g's i-th tile; false: there is none, or a wait expired
        bool ok = true;
        auto scores = [&](int g, int i) {
            const int t = ROWS ? i : 2 * i + g, item = 2 * t, s = item % P::RING;
            ok = ok && wait(TBAR_FULL + s, item / P::RING) && (!P::EARLY || i == 0 || wait(TBAR_READ + g, i - 1));
            if (!ok) return;
            if (meta[t & (P::META - 1)].at < 0) {
                ended[g] = true;
                return;
            }
            tc_after();
            if (elect_one()) {
                const u64 a = qd + (u32)((ROWS ? g : 0) * tb), bb = kd + (u32)(s * tb);
#pragma unroll
                for (int k = 0; k < KS; ++k)
                    mma_ss(tmem + P::S0 + g * kTile, a + ((k >> 2) * atom + 2 * (k & 3)), bb + ((k >> 2) * atom + 2 * (k & 3)), idesc_f16(kTile) | IDESC, k > 0);
                mma_commit(bar(TBAR_S + g));
                if (!ROWS || g == 1) mma_commit(bar(TBAR_EMPTY + s));
            }
            __syncwarp();
        };
        auto outputs = [&](int g, int i) {
            const int t = ROWS ? i : 2 * i + g, item = 2 * t + 1, s = item % P::RING;
            ok = ok && (ragged ? wait(TBAR_CLEAN + (t & (P::META - 1)), t / P::META) : wait(TBAR_FULL + s, item / P::RING));
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                ok = ok && wait(TBAR_P + 2 * g + half, i);
                if (!ok) return;
                tc_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 4 * half; k < 4 * half + 4; ++k)
                        mma_ts(tmem + P::O0 + g * P::OG, tmem + P::P0 + g * P::PG + 8 * k, vd + (u32)(s * tb + k * (16 * 128 / 16)), idesc_f16(DP) | IDESC | kIdescBAlongN,
                               k > 0 ? 1u : (u32)(i > 0));
                }
                __syncwarp();
            }
            if (P::EARLY || !ROWS || g == 1) {
                if (elect_one()) {
                    if (P::EARLY) mma_commit(bar(TBAR_O + g));
                    if (!ROWS || g == 1) mma_commit(bar(TBAR_EMPTY + s));
                }
                __syncwarp();
            }
        };
        ok = wait(TBAR_Q, 0);
        scores(0, 0);
        scores(1, 0);
        for (int i = 0; ok && !(ended[0] && ended[1]); ++i)
#pragma unroll
            for (int g = 0; g < 2; ++g)
                if (ok && !ended[g]) {
                    if (P::EARLY) scores(g, i + 1);
                    outputs(g, i);
                    if (!P::EARLY) scores(g, i + 1);
                }
        // The end of both groups: complete when every product is. After an expired wait too, products in flight end before TMEM is
        // freed.
        if (elect_one()) mma_commit(bar(TBAR_S)), mma_commit(bar(TBAR_S + 1)), mma_commit(bar(TBAR_END));
        __syncwarp();
        if (!ok) {
            volatile int never = 0;
            mbar_wait_suspended(bar(TBAR_END), 0, &never, &g_tcq_cross_error);
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    // Back to the launch's registers for the code that all warps share, behind the barrier: every softmax warp has had its larger share.
    if (warp < W_MMA) asm volatile("setmaxnreg.dec.sync.aligned.u32 168;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    if (warp == W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::COLS) : "memory");
    if (!parts) return;

    // ---- parts are added: those of the two groups where they share rows, those of a cluster's CTAs, each CTA a slice of the rows
    if (splits > 1) cluster_barrier();
    {
        constexpr int XP = (DP / 4) % 8 == 0 ? 7 : 3;
        const int rows = r1 - r0, s0 = rows * sp / splits, s1 = rows * (sp + 1) / splits, pieces = A.D / 8;
        for (int e = tid; e < (s1 - s0) * pieces; e += P::THREADS) {
            const int row = s0 + e / pieces, c8 = e % pieces;
            // four parts at a time, all of their loads under way at once
            constexpr int G = ROWS ? 1 : 2;
            float top = -INFINITY, acc[8] = {}, sum = 0.f;
            for (int k0 = 0; k0 < splits * G; k0 += 4) {
                float2 ml[4];
                float4 u[4], v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    ml[k] = make_float2(-INFINITY, 0.f), u[k] = v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (k0 + k < splits * G) {
                        const u32 p = peer_addr(sbase, (k0 + k) / G), at = ((k0 + k) % G) * kTile + row;
                        ml[k] = peer_ld2(p + P::ML0 + at * 8);
                        u[k] = peer_ld4(p + at * (DP * 4) + (((2 * c8) ^ (row & XP)) << 4)), v[k] = peer_ld4(p + at * (DP * 4) + (((2 * c8 + 1) ^ (row & XP)) << 4));
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float both = fmaxf(top, ml[k].x);
                    const float old = both == -INFINITY ? 1.f : ex2(top - both), f = part_factor(ml[k], both);
                    top = both;
                    sum = __fmaf_rn(ml[k].y, f, sum * old);
                    acc[0] = __fmaf_rn(u[k].x, f, acc[0] * old), acc[1] = __fmaf_rn(u[k].y, f, acc[1] * old);
                    acc[2] = __fmaf_rn(u[k].z, f, acc[2] * old), acc[3] = __fmaf_rn(u[k].w, f, acc[3] * old);
                    acc[4] = __fmaf_rn(v[k].x, f, acc[4] * old), acc[5] = __fmaf_rn(v[k].y, f, acc[5] * old);
                    acc[6] = __fmaf_rn(v[k].z, f, acc[6] * old), acc[7] = __fmaf_rn(v[k].w, f, acc[7] * old);
                }
            }
            const float f = sum != 0.f ? 1.f / sum : 0.f;
            u32 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = sum != 0.f ? weights2<DT>(acc[2 * j] * f, acc[2 * j + 1] * f) : 0u;
            u16* dst = A.out + row_at(A, b, h, r0 + row, (i64)A.T * A.heads * A.D, (i64)A.heads * A.D) + 8 * c8;
            *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    if (splits > 1) cluster_barrier();                        // a part may be read until here
}

template <int DT, int DP, bool ROWS>
int launch_tiles(const CrossArgs& A, const TileMaps& maps, void* stream) {
    typedef Tiles<DP, ROWS> P;
    const auto kern = k_cross_tiles<DT, DP, ROWS>;
    const int most = ROWS ? 2 * kTile : kTile;
    TilesPlan R = {};
    R.row_tiles = (A.rows + most - 1) / most;
    R.tile_rows = (((A.rows + R.row_tiles - 1) / R.row_tiles) + 31) & ~31;         // even shares, in warps
    const i64 units = (i64)A.B * A.kv_heads * R.row_tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(P::THREADS);
    cfg.dynamicSmemBytes = P::BYTES;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    // what a device can hold of clusters of 1 .. 8 CTAs, asked once per device
    static std::atomic<int> held[64][9];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return TCQ_ERR_DEVICE;
    if (!held[dev][1].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P::BYTES) != cudaSuccess) return TCQ_ERR_LAUNCH;
        // the register shares of the roles are taken from what the launch gives the CTA: less would leave them waiting
        cudaFuncAttributes fa;
        if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess) return TCQ_ERR_LAUNCH;
        if (fa.numRegs != P::LAUNCH_REGS) return TCQ_ERR_BUILD;
        for (int s = 8; s >= 1; --s) {
            int n = 0;
            cfg.gridDim = dim3(s);
            attr[0].val.clusterDim.x = s;
            cfg.numAttrs = 1;
            if (s == 1) n = tcq_sm_count();
            else if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) n = 0, cudaGetLastError();
            held[dev][s].store(n, std::memory_order_release);
        }
    }
    // Units that do not fill the device share their tiles among the CTAs of a cluster: the split with the least rounds of
    // tiles, at least two tiles to a group of a CTA.
    int splits = 1;
    const i64 tiles = ((i64)A.N + kTile - 1) / kTile;
    if (units < held[dev][1].load(std::memory_order_relaxed)) {
        double best = 1e30;
        for (int s = 1; s <= 8 && (s == 1 || (ROWS ? 2 : 4) * s <= tiles); ++s) {
            const int n = held[dev][s].load(std::memory_order_relaxed);
            if (n <= 0) continue;
            const double cost = (double)((units + n - 1) / n) / s * (1 + 0.02 * (s - 1));
            if (cost < best) best = cost, splits = s;
        }
    }
    if (units * splits > 0x7fffffff) return TCQ_ERR_SHAPE;
    R.splits = splits;
    R.by_tiles = make_fastdiv((unsigned)R.row_tiles), R.by_heads = make_fastdiv((unsigned)A.kv_heads), R.by_splits = make_fastdiv((unsigned)splits);
    cfg.gridDim = dim3((unsigned)(units * splits));
    attr[0].val.clusterDim.x = splits;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, A, maps, R) == cudaSuccess ? TCQ_OK : TCQ_ERR_LAUNCH;
}

// Zeros for queries without states (N = 0).
__global__ void __launch_bounds__(256) k_cross_none(uint4* out, i64 n) {
    pdl_launch_dependents();
    pdl_wait();
    for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < n; i += (i64)gridDim.x * 256) out[i] = make_uint4(0, 0, 0, 0);
}

// (D, N, kv_heads, B) of a 16-bit tensor with boxes of 64 elements of `box` states of one head.
bool encode(CUtensorMap* map, const void* p, int dtype, int D, int N, int heads, int B, i64 st, i64 sb, int box) {
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    // a dimension of size one has no stride of its own
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)N, (cuuint64_t)heads, (cuuint64_t)(sb ? B : 1)};
    const cuuint64_t row = (cuuint64_t)heads * D * 2, strides[3] = {N > 1 ? (cuuint64_t)st * 2 : row, (cuuint64_t)D * 2, sb ? (cuuint64_t)sb * 2 : row};
    const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, step[4] = {1, 1, 1, 1};
    return fn(map, dtype == TCQ_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(p), dims, strides,
              boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, int DP, int MT>
int launch_rows(const CrossArgs& A, const CUtensorMap& km, const CUtensorMap& vm, void* stream) {
    typedef Rows<DP, MT> P;
    const auto kern = k_cross_rows<DT, DP, MT>;
    RowsPlan R = {};
    // As many warps to a unit as its rows want, up to four. Up to head width 64, of those block heights the one that leaves the fewest warps
    // without rows (272 rows of each of 256 units over 160 states: nine blocks of 32 rows 17.1 us, three of 128 20.3); wider heads of many
    // units want every state read for as many rows as there are (33 rows of 512 units over 640 states of 128: three blocks of 16 73 us,
    // one of 64 48; of 8 units over 160 states 5.4 and 9.1).
    while (R.wm_log2 < 2 && (P::ROWS << R.wm_log2) < A.rows) ++R.wm_log2;
    if (DP <= 64 || (i64)A.B * A.kv_heads <= tcq_sm_count())
        for (int w = R.wm_log2 - 1, fewest = (A.rows + (P::ROWS << R.wm_log2) - 1) / (P::ROWS << R.wm_log2) << R.wm_log2; w >= 0; --w) {
            const int warps = (A.rows + (P::ROWS << w) - 1) / (P::ROWS << w) << w;
            if (warps < fewest) fewest = warps, R.wm_log2 = w;
        }
    const int rings = kRowWarps >> R.wm_log2;
    R.row_blocks = (A.rows + (P::ROWS << R.wm_log2) - 1) / (P::ROWS << R.wm_log2);
    R.block_rows = (((A.rows + R.row_blocks - 1) / R.row_blocks) + P::ROWS - 1) & ~(P::ROWS - 1);
    const i64 units = (i64)A.B * A.kv_heads * R.row_blocks;
    if (units > 0x7fffffff / 16) return TCQ_ERR_SHAPE;
    const int chunks = (A.N + P::CHUNK - 1) / P::CHUNK, sms = tcq_sm_count();
    R.units = (int)units;
    // whole units where they are enough for a CTA on every SM
    R.whole = units >= (i64)sms * rings;
    R.splits = 1;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    // Clusters of sixteen CTAs that the device holds at a time, and one more; asked once per device.
    static std::atomic<int> sixteens[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return TCQ_ERR_DEVICE;
    if (!sixteens[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P::bytes(kRowWarps, 3)) != cudaSuccess) return TCQ_ERR_LAUNCH;
        int n = 0;
        cfg.gridDim = dim3(16);
        cfg.dynamicSmemBytes = P::bytes(kRowWarps, 3);
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 16, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess)
            n = 0, cudaGetLastError();
        sixteens[dev].store(n + 1, std::memory_order_release);
    }
    // Else a unit's states are divided while there are SMs to spare and a ring keeps more chunks than adding its parts is worth: four, and one
    // for every eight rows. Into sixteen only where all those clusters run at once (one token over 16411 states, 8 key heads of 64: one
    // sequence, 8 clusters, 13.6 -> 10.8 us; four sequences 26 us with eight CTAs to a cluster, 37 with sixteen).
    if (!R.whole)
        while (R.splits < (units < sixteens[dev].load(std::memory_order_relaxed) && units * 16 <= sms ? 16 : 8) && units * R.splits < 2 * sms &&
               chunks >= rings * R.splits * (4 + R.block_rows / 8))
            R.splits *= 2;
    const int each = R.whole ? chunks : (chunks + rings * R.splits - 1) / (rings * R.splits);
    const int most = rings == 1 ? P::MOST : 3;
    R.stages = each + 1 < most ? each + 1 : most;
    R.by_blocks = make_fastdiv((unsigned)R.row_blocks), R.by_heads = make_fastdiv((unsigned)A.kv_heads);
    R.by_splits = make_fastdiv((unsigned)R.splits), R.by_workers = make_fastdiv((unsigned)(R.splits * rings));
    cfg.gridDim = dim3((unsigned)(R.whole ? (units + rings - 1) / rings : units * R.splits));
    cfg.dynamicSmemBytes = P::bytes(rings, R.stages);
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = R.splits, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = R.splits > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, A, km, vm, R) == cudaSuccess ? TCQ_OK : TCQ_ERR_LAUNCH;
}

// Call f(integral_constant<int, DP>) for the head width rounded up to one that is built.
template <class F>
int by_width(int d, F f) {
    if (d <= 32) return f(std::integral_constant<int, 32>());
    if (d <= 48) return f(std::integral_constant<int, 48>());
    if (d <= 64) return f(std::integral_constant<int, 64>());
    if (d <= 80) return f(std::integral_constant<int, 80>());
    if (d <= 96) return f(std::integral_constant<int, 96>());
    return f(std::integral_constant<int, 128>());
}

// Whether one of `batches` x n rows of w bytes, the first at `from`, sb from batch to batch and st from row to row (none negative), has
// a byte in [0, all). The batches are looked at one by one only where the rows' whole extent reaches into it.
bool rows_meet(i64 from, i64 all, i64 batches, i64 sb, int n, i64 st, i64 w) {
    const auto extent_meets = [&](i64 a, i64 length) { return a < all && a + length > 0; };
    if (!extent_meets(from, (batches - 1) * sb + (n - 1) * st + w)) return false;
    for (i64 i = 0; i < batches && from < all; ++i, from += sb) {
        if (!extent_meets(from, (n - 1) * st + w)) continue;
        // the first row that ends behind 0
        const i64 j = from + w > 0 || st == 0 ? 0 : (-from - w) / st + 1;
        if (j < n && extent_meets(from + j * st, w)) return true;
        if (sb == 0) break;
    }
    return false;
}

// Products of 16 rows or tiles of 128? A tile's CTA costs about 5 us before and behind its states, and computes 128 or 256 rows whatever
// there are; a row costs three times as much in the other kernel. Where tiles give every unit an SM of its own (and its states
// are divided over a cluster), they win from 256 states on if the rows are not few (us, products of 16 / tiles, heads of 64: 8 units
// of 33 rows over 160 states 6.5 / 6.3, over 640 12.7 / 8.8; of 17 rows 7.8 / 8.5; heads of 128: 33 rows over 640 8.4 / 11.0, 64
// rows 12.8 / 11.8; 64 units of 17 rows over 1280 17.4 / 12.7). Else by what the states of a unit cost in either, in picoseconds of
// the device (heads of 64: 1.15 a row and state against 0.35, 50,000 a tile of rows; of 128: 1.95, 0.43, 60,000): 512 units of 64
// rows over 640 states 27.8 / 37.3, over 2560 98.4 / 83.0; of 256 rows over 160 states 34 / 38, over 320 55 / 44; heads of 128, 256
// rows over 160 states 58 / 48.
bool prefer_tiles(i64 rows, int N, int D, i64 units) {
    const bool wide = D > 64;
    if (N < (wide ? 128 : 256)) return false;
    const i64 row_tiles = (rows + 255) / 256;
    if (units * row_tiles <= tcq_sm_count()) return N >= 256 && (rows > (wide ? 48 : 32) || (wide && rows > 16 && units * N >= 65536));
    const i64 small = !wide && rows > 16 ? (rows + 31) / 32 * 32 : (rows + 15) / 16 * 16, padded = rows <= 128 ? 128 : 256 * row_tiles;
    return (double)N * (wide ? 1.95 * (double)small - 0.43 * (double)padded : 1.15 * (double)small - 0.35 * (double)padded) > (wide ? 60000.0 : 50000.0) * (double)row_tiles;
}

}  // namespace

extern "C" {

int tcq_cross_attention(const void* q, int64_t q_sb, int64_t q_st, const void* k, int64_t k_sb, int64_t k_st, const void* v, int64_t v_sb,
                        int64_t v_st, int dtype, void* out, const int32_t* lens, const uint8_t* mask, int64_t mask_sb, float scale, int B,
                        int S, int T, int N, int heads, int kv_heads, int head_dim, void* stream) {
    if (!q || !out || (N > 0 && (!k || !v))) return TCQ_ERR_ARG;
    if (dtype != TCQ_DT_BF16 && dtype != TCQ_DT_F16) return TCQ_ERR_DTYPE;
    if (B < 1 || S < 1 || T < 1 || N < 0 || kv_heads < 1 || heads < 1 || heads % kv_heads) return TCQ_ERR_SHAPE;
    if (head_dim < 8 || head_dim > 128 || head_dim % 8) return TCQ_ERR_SHAPE;
    const i64 rows = (i64)S * T * (heads / kv_heads);
    if (rows > (1 << 30) || (i64)B * kv_heads > 0x7fffffff || N > (1 << 30)) return TCQ_ERR_SHAPE;
    if (!tcq_aligned(q, 16) || !tcq_aligned(k, 16) || !tcq_aligned(v, 16) || !tcq_aligned(out, 16)) return TCQ_ERR_ALIGN;
    if ((q_sb | q_st | k_sb | k_st | v_sb | v_st) & 7) return TCQ_ERR_ALIGN;
    if (k_sb < 0 || k_st < 0 || v_sb < 0 || v_st < 0 || (N > 1 && (k_st < 8 || v_st < 8))) return TCQ_ERR_ARG;
    // out may be q itself (a row's queries are read before it is written); beyond that it shares no byte with what is read
    const i64 width = (i64)heads * head_dim, all = (i64)B * S * T * width, row = (i64)kv_heads * head_dim;
    const auto meets = [&](const void* p, i64 batches, i64 sb, int n, i64 st, i64 w, int size = 2) {
        return rows_meet((intptr_t)p - (intptr_t)out, 2 * all, batches, sb * size, n, st * size, w * size);
    };
    const bool same = q == out && (T == 1 || q_st == width) && ((i64)B * S == 1 || q_sb == T * width);
    if (!same && q_sb >= 0 && q_st >= 0 && meets(q, (i64)B * S, q_sb, T, q_st, width)) return TCQ_ERR_ARG;
    if (N > 0 && (meets(k, B, k_sb, N, k_st, row) || meets(v, B, v_sb, N, v_st, row))) return TCQ_ERR_ARG;
    if (N > 0 && ((lens && meets(lens, 1, 0, 1, 0, B, 4)) || (mask && mask_sb >= 0 && meets(mask, B, mask_sb, 1, 0, N, 1)))) return TCQ_ERR_ARG;
    if (N == 0) {
        const i64 n = (i64)B * S * T * heads * head_dim / 8;
        const i64 blocks = (n + 255) / 256, most = (i64)tcq_sm_count() * 8;
        return launch_pdl(k_cross_none, dim3((unsigned)(blocks < most ? blocks : most)), 256, 0, stream, (uint4*)out, n);
    }
    // sequences that share one batch of states (stride 0) have one in the tensor map
    if (B == 1) k_sb = v_sb = 0;
    const auto maps_of = [&](CUtensorMap& km, CUtensorMap& vm, int box) {
        return encode(&km, k, dtype, head_dim, N, kv_heads, B, k_st, k_sb, box) && encode(&vm, v, dtype, head_dim, N, kv_heads, B, v_st, v_sb, box);
    };
    const int group = heads / kv_heads;
    const CrossArgs A = {(const u16*)q, q_sb, q_st, (u16*)out, lens, mask, mask_sb, B, S, T, N, heads, kv_heads, group, head_dim, (int)rows,
                         k_sb != 0, v_sb != 0, make_fastdiv((unsigned)group), make_fastdiv((unsigned)T), scale * 1.4426950408889634f};
    if (prefer_tiles(rows, N, head_dim, (i64)B * kv_heads)) {
        TileMaps maps;
        if (!maps_of(maps.k, maps.v, kTile) || (mask && !maps_of(maps.k_half, maps.v_half, kTile / 2))) return TCQ_ERR_DEVICE;
        if (!mask) maps.k_half = maps.k, maps.v_half = maps.v;
        return by_width(head_dim, [&](auto d) {
            constexpr int DP = decltype(d)::value;
            if (dtype == TCQ_DT_BF16) return rows <= kTile ? launch_tiles<TCQ_DT_BF16, DP, false>(A, maps, stream) : launch_tiles<TCQ_DT_BF16, DP, true>(A, maps, stream);
            return rows <= kTile ? launch_tiles<TCQ_DT_F16, DP, false>(A, maps, stream) : launch_tiles<TCQ_DT_F16, DP, true>(A, maps, stream);
        });
    }
    return by_width(head_dim, [&](auto d) {
        constexpr int DP = decltype(d)::value;
        CUtensorMap km, vm;
        if (!maps_of(km, vm, Rows<DP, 1>::CHUNK)) return (int)TCQ_ERR_DEVICE;
        if constexpr (DP <= 64) {
            if (rows > 16) return dtype == TCQ_DT_BF16 ? launch_rows<TCQ_DT_BF16, DP, 2>(A, km, vm, stream) : launch_rows<TCQ_DT_F16, DP, 2>(A, km, vm, stream);
        }
        return dtype == TCQ_DT_BF16 ? launch_rows<TCQ_DT_BF16, DP, 1>(A, km, vm, stream) : launch_rows<TCQ_DT_F16, DP, 1>(A, km, vm, stream);
    });
}

}  // extern "C"
