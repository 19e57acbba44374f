// Attention to an encoder's states of another length: out = softmax(scale q k^T) v over the states that are there.
//
// q (B S, T, heads D): the S batches b S .. b S + S - 1 read the states of sequence b; k, v (B, N, kv_heads D); lens (B) and a mask
// (B, N) say which states are there. The rows that read one key head of one sequence are its R = S T group queries, token by
// token, `group` heads to a token: they share every load of K and V.
#include "memory.cuh"
#include "tma.cuh"

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

TCQ_HD float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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

// Weights are 2^(x - m + kRef), m the row's reference, moved only when a score passes it by more than kSlack: below 2^13, so
// that FP16 holds them with 11 bits from there down to 2^-14.
constexpr float kRef = 5.f, kSlack = 8.f;

// ------------------------------------------------------------------------------------------------ products of 16 rows
// Warps of 16 query rows on m16n8k16 products, for few rows or few states: bound by HBM where the states are many, by latency where
// they are few. A CTA of eight warps takes WM groups of 16 rows and divides the keys among its 8 / WM key groups, and those
// of a cluster of CTAs: each key group streams chunks of 32 states (16 above head width 64) through a ring of its own (TMA, 128-byte swizzle, zeros past D and N).
// The first warp of a key group requests them and skips chunks of which the mask leaves nothing. The parts of a row are
// added in shared memory, a cluster's through distributed shared memory, always in the same order.
constexpr int kRowWarps = 8;

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
template <int DP>
struct Rows {
    static constexpr int CHUNK = DP <= 64 ? 32 : 16;                                                 // states
    static constexpr int ATOMS = (DP + 63) / 64, HALF = ATOMS * CHUNK * 128, STAGE = 2 * HALF;       // bytes of a chunk's keys, of both
    static constexpr int PITCH = DP + 4;                                                             // floats of a part's row
    static constexpr int PARTS = kRowWarps * 16 * PITCH * 4;
    static constexpr int bytes(int rings, int stages) {                                             // 3 stages of 8 rings: 197 KB
        const int ring = rings * stages * STAGE;
        return (ring > PARTS ? ring : PARTS) + rings * stages * 24 + 16;
    }
};

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ u32 peer_addr(u32 addr, u32 rank) {
    u32 r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float peer_ld(u32 addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 peer_ld2(u32 addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

template <int DT, int DP>
__global__ void __launch_bounds__(kRowWarps * 32, DP <= 64 ? 2 : 1)
k_cross_rows(const CrossArgs A, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int wm_log2, int stages,
             int splits, int row_blocks, int block_rows) {
    typedef Rows<DP> P;
    constexpr int KS = DP / 16, NT = DP / 8, kChunk = P::CHUNK, NK = kChunk / 8;
    constexpr u32 kAll = (u32)((1ull << kChunk) - 1);
    extern __shared__ __align__(1024) char smem_rows[];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int WM = 1 << wm_log2, rings = kRowWarps >> wm_log2, wm = warp & (WM - 1), kg = warp >> wm_log2;
    const u32 sbase = smem_u32(smem_rows);
    const int ring_bytes = max(rings * stages * P::STAGE, P::PARTS);
    const u32 bars = sbase + ring_bytes;                           // full, empty of each stage of each ring
    int2* meta = reinterpret_cast<int2*>(smem_rows + ring_bytes + rings * stages * 16);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_rows + ring_bytes + rings * stages * 24);
    auto full = [&](int s) -> u32 { return bars + 16 * (kg * stages + s); };
    auto empty = [&](int s) -> u32 { return bars + 16 * (kg * stages + s) + 8; };
    if (tid < rings * stages) {
        mbar_init(bars + 16 * tid, 1);
        mbar_init(bars + 16 * tid + 8, WM);
        if (tid == 0) *abort_flag = 0;
        mbar_init_fence();
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();

    const int rank = blockIdx.x % splits, unit = blockIdx.x / splits, rb = unit % row_blocks, bh = unit / row_blocks;
    const int b = bh / A.kv_heads, h = bh - b * A.kv_heads, r0 = rb * block_rows, r1 = min(A.rows, r0 + block_rows);
    const int len = states_of(A, b);
    // this key group's chunks [c0, c1)
    const int chunks = (len + kChunk - 1) / kChunk, worker = rank * rings + kg, workers = splits * rings;
    const int c0 = (int)((i64)chunks * worker / workers), c1 = (int)((i64)chunks * (worker + 1) / workers);

    // ---- the producer: the next chunk that holds a state, its truth values as bits
    const unsigned char* mrow = A.mask ? A.mask + b * A.mask_sb : nullptr;
    int pc = c0, ps = 0, puse = 0;
    unsigned char pm = 0;
    auto look = [&]() {                                            // request the mask of chunk pc
        if (mrow && pc < c1) pm = lane < kChunk && pc * kChunk + lane < len ? mrow[pc * kChunk + lane] : 0;
    };
    bool pend = false;
    auto issue = [&]() {
        if (pend) return;
        u32 bits = 0;
        int at = -1;
        while (pc < c1) {
            const int n = len - pc * kChunk;
            bits = mrow ? __ballot_sync(0xffffffffu, pm != 0) : n >= kChunk ? kAll : (1u << n) - 1u;
            at = pc++;
            look();
            if (bits) break;
        }
        if (!bits) at = -1, pend = true;
        if (puse && !mbar_wait_suspended(empty(ps), (puse - 1) & 1, abort_flag, &g_tcq_cross_error)) pend = true, at = -1;
        if (lane == 0) {
            meta[kg * stages + ps] = make_int2(at, (int)bits);
            if (at < 0) {
                mbar_arrive(full(ps));
            } else {
                const u32 dst = sbase + (kg * stages + ps) * P::STAGE;
                mbar_expect_tx(full(ps), P::STAGE);
#pragma unroll
                for (int a = 0; a < P::ATOMS; ++a) {
                    tma_load_4d(dst + a * (kChunk * 128), &kmap, full(ps), 64 * a, at * kChunk, h, b * A.kb);
                    tma_load_4d(dst + P::HALF + a * (kChunk * 128), &vmap, full(ps), 64 * a, at * kChunk, h, b * A.vb);
                }
            }
        }
        __syncwarp();
        if (++ps == stages) ps = 0, ++puse;
    };
    const bool live = r0 + 16 * wm < r1;                           // a warp without a row only keeps the barriers going
    if (wm == 0) {
        look();
        for (int i = 0; i + 1 < stages; ++i) issue();
    }

    // ---- this warp's 16 rows: g and g + 8
    u32 q[KS][4];
    {
        const int ra = r0 + 16 * wm + g, rc = ra + 8;
        const u16* qa = A.q + row_at(A, b, h, min(ra, A.rows - 1), A.q_sb, A.q_st);
        const u16* qc = A.q + row_at(A, b, h, min(rc, A.rows - 1), A.q_sb, A.q_st);
        const u32 flip = A.scale_log2 < 0.f ? 0x80008000u : 0u;    // a negative scale turns the queries
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = 16 * k + 8 * e + 2 * t;
                const bool in = DP % 16 == 0 && d < A.D;
                q[k][2 * e] = in && ra < r1 ? *reinterpret_cast<const u32*>(qa + d) ^ flip : 0u;
                q[k][2 * e + 1] = in && rc < r1 ? *reinterpret_cast<const u32*>(qc + d) ^ flip : 0u;
            }
    }
    const float c = fabsf(A.scale_log2);
    float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    // One chunk: 32 scores of each row, weights, O += P V. Matrices of 8 x 8 are read from the swizzled tiles: 16-byte piece p of row r
    // lies at p ^ (r & 7).
    auto chunk = [&](auto masked_c, u32 bits, u32 kt, u32 vt) {
        constexpr bool MASKED = decltype(masked_c)::value;
        float s[NK][4];
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
            const int r = 8 * n + (lane & 7);
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
                u32 f[4];
                const int p = 2 * k + (lane >> 3);                 // pieces of 8 elements: two of step k, two of step k + 1
                ldsm4(kt + (p >> 3) * (kChunk * 128) + r * 128 + (((p & 7) ^ (r & 7)) << 4), f);
                mma16816<DT>(s[n], q[k][0], q[k][1], q[k][2], q[k][3], f[0], f[1]);
                if (k + 1 < KS) mma16816<DT>(s[n], q[k + 1][0], q[k + 1][1], q[k + 1][2], q[k + 1][3], f[2], f[3]);
            }
        }
        if (MASKED) {
            const u32 w = bits >> (2 * t);
#pragma unroll
            for (int n = 0; n < NK; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (!(w >> (8 * n + e) & 1)) s[n][e] = s[n][2 + e] = -INFINITY;
        }
        float top[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            top[e] = fmaxf(s[0][2 * e], s[0][2 * e + 1]);
#pragma unroll
            for (int n = 1; n < NK; ++n) top[e] = fmaxf(top[e], fmaxf(s[n][2 * e], s[n][2 * e + 1]));
        }
        if (MASKED) {                                              // c may be zero: -inf stays -inf
            top[0] = top[0] == -INFINITY ? top[0] : top[0] * c;
            top[1] = top[1] == -INFINITY ? top[1] : top[1] * c;
        } else {
            top[0] *= c, top[1] *= c;
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
                const bool move = top[e] > m[e] + kSlack;
                f[e] = move ? ex2(m[e] - top[e]) : 1.f;
                if (move) m[e] = top[e];
                l[e] *= f[e];
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) o[i][0] *= f[0], o[i][1] *= f[0], o[i][2] *= f[1], o[i][3] *= f[1];
        }
        const float base[2] = {kRef - (m[0] == -INFINITY ? 0.f : m[0]), kRef - (m[1] == -INFINITY ? 0.f : m[1])};
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = MASKED && s[n][e] == -INFINITY ? -INFINITY : __fmaf_rn(s[n][e], c, base[e >> 1]);
                s[n][e] = ex2(x);
            }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < NK; ++n) sum += s[n][2 * e] + s[n][2 * e + 1];
            l[e] += sum;
        }
#pragma unroll
        for (int k = 0; k < NK / 2; ++k) {
            const u32 a0 = pack2<DT>(s[2 * k][0], s[2 * k][1]), a1 = pack2<DT>(s[2 * k][2], s[2 * k][3]), a2 = pack2<DT>(s[2 * k + 1][0], s[2 * k + 1][1]),
                      a3 = pack2<DT>(s[2 * k + 1][2], s[2 * k + 1][3]);
            // what lies where no state is may be anything, NaN too: this lane's keys 16 k + 2 t, + 1 and 8 further
            u32 z0 = 0xffffffffu, z1 = 0xffffffffu;
            if (MASKED) {
                const u32 w = bits >> (16 * k + 2 * t);
                z0 = (w & 1 ? 0xffffu : 0u) | (w & 2 ? 0xffff0000u : 0u);
                z1 = (w & 256 ? 0xffffu : 0u) | (w & 512 ? 0xffff0000u : 0u);
            }
            const int r = 16 * k + (lane & 15);
#pragma unroll
            for (int i = 0; i < NT; i += 2) {
                u32 f[4];
                const int p = i + (lane >> 4);
                ldsm4t(vt + (p >> 3) * (kChunk * 128) + r * 128 + (((p & 7) ^ (r & 7)) << 4), f);
                mma16816<DT>(o[i], a0, a1, a2, a3, MASKED ? f[0] & z0 : f[0], MASKED ? f[1] & z1 : f[1]);
                mma16816<DT>(o[i + 1], a0, a1, a2, a3, MASKED ? f[2] & z0 : f[2], MASKED ? f[3] & z1 : f[3]);
            }
        }
    };
    int slot = 0, use = 0;
    for (;;) {
        if (!mbar_wait_suspended(full(slot), use & 1, abort_flag, &g_tcq_cross_error)) break;
        const int2 what = meta[kg * stages + slot];
        if (what.x < 0) break;
        if (wm == 0) issue();                                      // into the stage that was used last
        const u32 kt = sbase + (kg * stages + slot) * P::STAGE, vt = kt + P::HALF;
        if (live) {
            if ((u32)what.y == kAll) chunk(std::false_type(), kAll, kt, vt);
            else chunk(std::true_type(), (u32)what.y, kt, vt);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(slot));
        if (++slot == stages) slot = 0, ++use;
    }
    if (wm == 0 && *abort_flag) {                                  // copies on their way land before their stages are left
        volatile int never = 0;
        for (; use < puse || (use == puse && slot < ps); use += slot + 1 == stages, slot = slot + 1 == stages ? 0 : slot + 1)
            mbar_wait_suspended(full(slot), use & 1, &never, &g_tcq_cross_error, kWaitNs / 20);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    if (rings * splits == 1) {
        if (!live) return;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = r0 + 16 * wm + g + 8 * e;
            if (r >= r1) continue;
            const float f = l[e] != 0.f ? 1.f / l[e] : 0.f;
            u32* dst = reinterpret_cast<u32*>(A.out + row_at(A, b, h, r, (i64)A.T * A.heads * A.D, (i64)A.heads * A.D));
#pragma unroll
            for (int i = 0; i < NT; ++i)
                if (8 * i < A.D) dst[4 * i + t] = pack2<DT>(o[i][2 * e] * f, o[i][2 * e + 1] * f);
        }
        return;
    }
    // ---- parts to shared memory (every chunk has arrived), added by all warps: rows of the CTA, one pair of elements a thread
    __syncthreads();
    float* part = reinterpret_cast<float*>(smem_rows) + (size_t)warp * 16 * P::PITCH;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        float* row = part + (g + 8 * e) * P::PITCH;
#pragma unroll
        for (int i = 0; i < NT; ++i) *reinterpret_cast<float2*>(row + 8 * i + 2 * t) = make_float2(o[i][2 * e], o[i][2 * e + 1]);
        if (t == 0) row[DP] = m[e], row[DP + 1] = l[e];
    }
    if (splits > 1) cluster_barrier();
    else __syncthreads();
    const int rows = r1 - r0, f0 = rows * rank / splits, f1 = rows * (rank + 1) / splits, half = A.D / 2;
    for (int i = tid; i < (f1 - f0) * half; i += kRowWarps * 32) {
        const int rr = f0 + i / half, d = 2 * (i % half), w = rr >> 4;
        const u32 at = sbase + (((u32)w * 16 + (rr & 15)) * P::PITCH) * 4;
        float top = -INFINITY;
        for (int k = 0; k < splits; ++k) {
            const u32 p = peer_addr(at, k);
            for (int j = 0; j < rings; ++j) top = fmaxf(top, peer_ld(p + (j * WM * 16 * P::PITCH + DP) * 4));
        }
        float sum = 0.f, a0 = 0.f, a1 = 0.f;
        for (int k = 0; k < splits; ++k) {
            const u32 p = peer_addr(at, k);
            for (int j = 0; j < rings; ++j) {
                const u32 pj = p + j * WM * 16 * P::PITCH * 4;
                const float2 ml = peer_ld2(pj + DP * 4), v = peer_ld2(pj + d * 4);
                const float f = top == -INFINITY ? (ml.y == ml.y ? 0.f : 1.f) : ex2(ml.x - top);
                // a part without weight adds nothing, unless its sum is NaN: the row has to say so
                if (f == 0.f && ml.y == ml.y) continue;
                sum = __fmaf_rn(ml.y, f, sum), a0 = __fmaf_rn(v.x, f, a0), a1 = __fmaf_rn(v.y, f, a1);
            }
        }
        const float f = sum != 0.f ? 1.f / sum : 0.f;
        *reinterpret_cast<u32*>(A.out + row_at(A, b, h, r0 + rr, (i64)A.T * A.heads * A.D, (i64)A.heads * A.D) + d) = pack2<DT>(a0 * f, a1 * f);
    }
    if (splits > 1) cluster_barrier();                             // a part may be read until here
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

template <int DT, int DP>
int launch_rows(const CrossArgs& A, const CUtensorMap& km, const CUtensorMap& vm, void* stream) {
    typedef Rows<DP> P;
    const auto kern = k_cross_rows<DT, DP>;
    int wm = 0;
    while (wm < 3 && (16 << wm) < A.rows) ++wm;
    const int rings = kRowWarps >> wm, row_blocks = (A.rows + (16 << wm) - 1) / (16 << wm);
    const int block_rows = (((A.rows + row_blocks - 1) / row_blocks) + 15) & ~15;
    const i64 units = (i64)A.B * A.kv_heads * row_blocks;
    const int chunks = (A.N + P::CHUNK - 1) / P::CHUNK, sms = tcq_sm_count();
    int splits = 1;
    while (splits < 8 && units * splits < 2 * sms && chunks >= 2 * rings * splits * 2) splits *= 2;
    const int each = (chunks + rings * splits - 1) / (rings * splits);
    const int stages = each + 1 < 3 ? each + 1 : 3;
    if (units * splits > 0x7fffffff) return TCQ_ERR_SHAPE;
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return TCQ_ERR_DEVICE;
    if (!(set.load(std::memory_order_relaxed) >> dev & 1)) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P::bytes(kRowWarps, 3)) != cudaSuccess)
            return TCQ_ERR_LAUNCH;
        set.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * splits));
    cfg.blockDim = dim3(kRowWarps * 32);
    cfg.dynamicSmemBytes = P::bytes(rings, stages);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, A, km, vm, wm, stages, splits, row_blocks, block_rows) == cudaSuccess ? TCQ_OK : TCQ_ERR_LAUNCH;
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
    if (N == 0) {
        const i64 n = (i64)B * S * T * heads * head_dim / 8;
        const i64 blocks = (n + 255) / 256, most = (i64)tcq_sm_count() * 8;
        return launch_pdl(k_cross_none, dim3((unsigned)(blocks < most ? blocks : most)), 256, 0, stream, (uint4*)out, n);
    }
    // sequences that share one batch of states (stride 0) have one in the tensor map
    if (B == 1) k_sb = v_sb = 0;
    CUtensorMap km, vm;
    const int box = by_width(head_dim, [](auto d) { return Rows<decltype(d)::value>::CHUNK; });
    if (!encode(&km, k, dtype, head_dim, N, kv_heads, B, k_st, k_sb, box) || !encode(&vm, v, dtype, head_dim, N, kv_heads, B, v_st, v_sb, box))
        return TCQ_ERR_DEVICE;
    const int group = heads / kv_heads;
    const CrossArgs A = {(const u16*)q, q_sb, q_st, (u16*)out, lens, mask, mask_sb, B, S, T, N, heads, kv_heads, group, head_dim, (int)rows,
                         k_sb != 0, v_sb != 0, make_fastdiv((unsigned)group), make_fastdiv((unsigned)T), scale * 1.4426950408889634f};
    return by_width(head_dim, [&](auto d) {
        constexpr int DP = decltype(d)::value;
        return dtype == TCQ_DT_BF16 ? launch_rows<TCQ_DT_BF16, DP>(A, km, vm, stream) : launch_rows<TCQ_DT_F16, DP>(A, km, vm, stream);
    });
}

}  // extern "C"
