// Attention over the 8-bit cache.
#include <type_traits>

#include "memory.cuh"
#include "tc.cuh"

__device__ int g_tcq_attention_error;

int tcq_attention_error(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tcq_attention_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && v) {
        const int z = 0;
        if (cudaMemcpyToSymbol(g_tcq_attention_error, &z, sizeof(int)) != cudaSuccess) return -1;
    }
    return v;
}

namespace {

using namespace tcq;

TCQ_HD void out_of_range() { atomicOr(&g_tcq_attention_error, 2); }

// Tokens of a sequence, page of a block: clamped to what exists, an index out of range reported.
TCQ_HD int tokens_of(const int* lens, i64 b, int blocks) {
    const int n = lens[b], most = blocks * kBlk;
    if ((unsigned)n > (unsigned)most) {
        out_of_range();
        return n < 0 ? 0 : most;
    }
    return n;
}
TCQ_HD int queries_of(const int* count, i64 b, int T) {
    if (!count) return T;
    const int n = count[b];
    if ((unsigned)n > (unsigned)T) {
        out_of_range();
        return n < 0 ? 0 : T;
    }
    return n;
}
TCQ_HD int page_in(int p, int pages) {
    if ((unsigned)p >= (unsigned)pages) {
        out_of_range();
        return p < 0 ? 0 : pages - 1;
    }
    return p;
}
TCQ_HD int page_of(const int* row, int blk, int pages) { return page_in(row[blk], pages); }

// ------------------------------------------------------------------------------------------------ few query rows
// T * group <= 32 query rows share a key head (single tokens, short action sequences; 16 rows above head width 64): the kernel
// streams the pages once. Bound by HBM for long sequences (4 x 131037 keys of 8 heads of 64: 104 us, 5.1 TB/s), by the latency of a
// warp's page (about 1.5 us) for short ones (one token over 203 keys: 4.6 us a call).
//
// Mathematics. With integers k, v and block scales ks, vs: score x = (q . k) ks scale log2(e) + log2(vs), reference
// m >= x - 10.5, weight p = 2^(x - m + 5); out = sum p v / sum (p / vs). Folding vs into the exponent keeps every operand of a
// product an exact small integer or one rounding of p, and the sum of p is formed in FP32 before that rounding. m moves only
// when a score passes it by more than 10.5, so the accumulators are rarely rescaled. Operands are FP16, accumulators FP32: an
// int8 is exact, a query row is scaled by a power of two so that its largest element lies in [2^14, 2^15) (elements below 2^-28
// of it lose bits, those of BF16 inputs above that lose none), and p <= 2^15.5 keeps 11 bits down to 2^-19 of the reference's
// and is dropped below 2^-30 of it: with n keys a row is off by at most 2^-11 sum p |v| + 2^-30 n max |v| for it (p normed here;
// F16 outputs of two 4096-token prompts are 2.8e-4 from 64 bits, 2.1e-4 with FP32 weights). BF16 in its place would keep 8 bits of p.
//
// Layout. A warp takes whole pages. S^T = K Q^T and O^T = V^T P^T are m16n8k16 products with the 64 keys (or the D value
// rows) as rows and NT tiles of 8 queries as columns, so that one token's few queries waste least. The order of a contraction is
// free, so lane (n, t) reads 16 consecutive bytes of key row n (or of value row n: 16 tokens) and feeds them to four products:
// one 16-byte shared load per 16 elements and no transposition. Keys are assigned to the rows of S^T so that a lane's
// weights, turned by movmatrix, are exactly the tokens whose values it reads: row c = 2 t + e of block nb (8 rows) is
// key 16 t + 2 nb + e.
//
// int8 -> FP16: u = byte ^ 0x80, 0x6400 | u is 1024 + u, minus 1152: five instructions for four elements.

constexpr float kRef = 5.f;           // log2 of the weight of a score equal to the reference
constexpr float kSlack = 10.5f;       // growth of the maximum that does not move the reference: weights up to 2^15.5

TCQ_HD float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
TCQ_HD float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Value scales below 2^-90, zero (a block of zeros) among them: the block's values count as zero, and 2^-90 takes the scale's
// place in the exponent and the sum, so that its tokens keep their weight and the sum stays in range.
constexpr float kLeastScale = 8.0779357e-28f;
TCQ_HD float safe_scale(float vs) { return vs < kLeastScale ? kLeastScale : vs; }

TCQ_HD void int8x4_to_half(u32 w, u32& lo, u32& hi) {
    const u32 u = w ^ 0x80808080u, c = 0x64806480u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(__byte_perm(u, 0x64646464u, 0x4140)), "r"(c));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(__byte_perm(u, 0x64646464u, 0x4342)), "r"(c));
}
TCQ_HD u32 half2_of(float lo, float hi) { return pack2<TCQ_DT_F16>(lo, hi); }

TCQ_HD void mma16816(float (&d)[4], u32 a0, u32 a1, u32 a2, u32 a3, u32 b0, u32 b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An 8 x 8 matrix of 16-bit elements, a row in four lanes, transposed.
TCQ_HD u32 turned(u32 v) {
    u32 r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Power of two that brings a row whose largest magnitude is amax into FP16's upper range, and its inverse.
TCQ_HD float row_scale(float amax, float& back) {
    int e = (int)((__float_as_uint(amax) >> 23) & 255) - 127;           // floor(log2), -127 for zero and subnormals
    e = min(max(e, -100), 126);
    back = __uint_as_float((u32)(e - 14 + 127) << 23);
    return __uint_as_float((u32)(14 - e + 127) << 23);
}

struct AttnArgs {
    tcq_kv8_cache cache;
    const u16* q;
    i64 q_sb, q_st;
    u16* out;
    const int* table;
    const int* lens;
    const int* count;
    float* part;           // partial rows of segments that do not cover their unit
    int* counters;
    int blocks, causal, B, T, heads, group;
    FastDiv by_group;
    float scale_log2;      // scale * log2(e)
};

// Plan of the few-row kernel. Every warp has a ring of NH half pages (64 D bytes: a block's keys or its values) of its own. As
// many warps as their registers and rings allow: a warp alone issues one instruction in about four clocks (32 ragged sequences
// and 4 x 131037 keys: 39 and 107 us with 12 warps, 40 and 109 with 8; 16 spill registers: 50 and 125).
template <int D, int NT>
struct Few {
    static constexpr int HALF = kBlk * D;
    static constexpr int WARPS = NT == 1 ? (D < 128 ? 12 : 8) : NT == 2 && D <= 64 ? 12 : 8;
    static constexpr int FIT = 216 * 1024 / (WARPS * HALF), NH = FIT < 8 ? FIT : 8;
    static_assert(NH >= 3, "a half page in use and two on their way");
    static constexpr int HDR = WARPS * NH * HALF;                          // ks, vs of each half page
    static constexpr int SCAN = HDR + WARPS * NH * 8;                      // the block's scan of the lengths
    static constexpr int BYTES = SCAN + 4 * WARPS * (int)sizeof(int);
    static_assert(8 * NT * (D + 2) * 4 <= NH * HALF, "a warp's part of a unit fits its ring");
};

// 16-byte chunk c of key row r lies at chunk c ^ swap(r): rows of 128 bytes put their halves on alternating banks.
template <int D>
TCQ_HD int key_chunk(int r, int c) { return D == 128 ? c ^ ((r & 1) << 2) : c; }

// A position in the flattened list of pages: sequence b, key head h, unit (b, h) begins at ubeg and takes vp places, of which
// the first np are pages.
struct Place {
    int b, h, ubeg, vp, np;
};

// The part of a unit that worker w wrote: a worker has at most two, of its first unit and (as that unit's first worker) its last.
TCQ_HD i64 part_slot(int w, int first) { return 2 * (i64)w + (w == first ? 1 : 0); }

// One warp adds parts of a unit, those of workers from, from + step, .. to, in that order: to the unit's R output rows, or, with
// out NULL, to the part of worker `from`. Kept out of line, four parts at a time: its loads in flight want registers, and eight
// parts made the caller spill (107 -> 124 us at 4 x 131037 keys).
template <int DT, int D>
__device__ __noinline__ void add_parts(float* parts, i64 size, int first, int from, int to, int step, int R, int group, u16* out, i64 token) {
    constexpr int NI = 4, NB = 4;                 // pairs of elements of a lane, parts requested at once
    const int lane = threadIdx.x & 31;
    float* target = parts + part_slot(from, first) * size;
#pragma unroll 1
    for (int i0 = 0; i0 < R * (D / 2); i0 += 32 * NI) {
        float2 acc[NI] = {};
        float top[NI], sum[NI] = {};
        int off[NI], ml[NI];
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            const int i = min(i0 + lane + 32 * k, R * (D / 2) - 1), r = i / (D / 2);
            off[k] = r * (D + 2) + 2 * (i - r * (D / 2)), ml[k] = r * (D + 2) + D;
            top[k] = -INFINITY;
        }
#pragma unroll 1
        for (int w0 = from; w0 <= to; w0 += NB * step) {
            float2 v[NB][NI], e[NB][NI];
#pragma unroll
            for (int w = 0; w < NB; ++w) {
                const int at = w0 + w * step <= to ? w0 + w * step : w0;
                const float* part = parts + part_slot(at, first) * size;
#pragma unroll
                for (int k = 0; k < NI; ++k) {
                    v[w][k] = __ldcg(reinterpret_cast<const float2*>(part + off[k]));
                    e[w][k] = __ldcg(reinterpret_cast<const float2*>(part + ml[k]));
                }
            }
#pragma unroll
            for (int w = 0; w < NB; ++w)
                if (w0 + w * step <= to) {
#pragma unroll
                    for (int k = 0; k < NI; ++k) {
                        const float nt = fmaxf(top[k], e[w][k].x), keep = nt == -INFINITY ? 0.f : ex2(top[k] - nt),
                                    f = nt == -INFINITY ? 0.f : ex2(e[w][k].x - nt);
                        top[k] = nt;
                        sum[k] = __fmaf_rn(e[w][k].y, f, sum[k] * keep);
                        acc[k].x = __fmaf_rn(v[w][k].x, f, acc[k].x * keep), acc[k].y = __fmaf_rn(v[w][k].y, f, acc[k].y * keep);
                    }
                }
        }
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            const int i = i0 + lane + 32 * k, r = i / (D / 2), tq = r / group;
            if (i >= R * (D / 2)) continue;
            const float f = sum[k] != 0.f ? 1.f / sum[k] : 0.f;
            if (out) reinterpret_cast<u32*>(out + tq * token + (i64)(r - tq * group) * D)[i - r * (D / 2)] = pack2<DT>(acc[k].x * f, acc[k].y * f);
            else *reinterpret_cast<float2*>(target + off[k]) = acc[k];
        }
    }
    if (out) return;
    // references and sums last: every lane has read them by now
    float top = -INFINITY, sum = 0.f;
    if (lane < R)
        for (int w = from; w <= to; w += step) {
            const float2 e = __ldcg(reinterpret_cast<const float2*>(parts + part_slot(w, first) * size + lane * (D + 2) + D));
            const float nt = fmaxf(top, e.x);
            if (nt == -INFINITY) continue;
            sum = __fmaf_rn(e.y, ex2(e.x - nt), sum * ex2(top - nt));
            top = nt;
        }
    __syncwarp();
    if (lane < R) *reinterpret_cast<float2*>(target + lane * (D + 2) + D) = make_float2(top, sum);
}

// Work, by what the lengths say:
// - the pages of all sequences and heads form one list, cut into equal runs, one per warp (a unit is one head of one sequence;
//   an empty one takes a place without a page). A warp that holds a whole unit writes its output; parts of a unit go to the
//   workspace, and the last of its warps to arrive adds them in their order, so the result does not depend on timing;
// - no more units than CTAs, of at most three pages per warp: a CTA takes a unit, its warps every WARPS-th page, and the parts are
//   added in shared memory (one token over 203 keys of 8 heads: 4.9 us a call, through the workspace 10.8);
// - whole != 0 (many short sequences, told by the host): each warp takes whole units, one after the other.
template <int DT, int D, int NT>
__global__ void __launch_bounds__(Few<D, NT>::WARPS * 32, 1) k_attention_few(const AttnArgs A, int whole) {
    typedef Few<D, NT> P;
    constexpr int NH = P::NH, KS = D / 16, WARPS = P::WARPS;
    extern __shared__ __align__(16) char smem[];
    int* s_scan = reinterpret_cast<int*>(smem + P::SCAN);
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = lane >> 2, t = lane & 3;
    const int Hk = A.cache.kv_heads, R = A.T * A.group;
    // consecutive workers on different SMs
    const int me = warp * gridDim.x + blockIdx.x, workers = WARPS * gridDim.x;
    char* ring = smem + warp * NH * P::HALF;
    float2* hdr = reinterpret_cast<float2*>(smem + P::HDR) + warp * NH;

    // ---- this worker's places x0, x0 + stride, .. below x1, and the unit they begin in
    int chunk = 1, stride = 1, x0, x1;
    Place at;
    auto places = [&](int len) { return max(1, (len + kBlk - 1) / kBlk); };
    if (whole) {
        if (me >= A.B * Hk) return;
        at.b = me / Hk, at.h = me - at.b * Hk;
        x0 = 0, x1 = 1 << 30;
    } else {
        // all sequences' lengths: every thread a run of them, summed over the block
        const int per = (A.B + WARPS * 32 - 1) / (WARPS * 32), b0 = min(A.B, tid * per), b1 = min(A.B, b0 + per);
        int mine = 0, most = 0;
        for (int b = b0; b < b1; ++b) {
            const int v = places(tokens_of(A.lens, b, A.blocks));
            mine += v, most = max(most, v);
        }
        int scan = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) s_scan[warp] = scan;
        const bool block = A.B * Hk <= gridDim.x && __syncthreads_and(most <= 3 * WARPS);
        if (A.B * Hk > gridDim.x) __syncthreads();
        if (block) {
            if (blockIdx.x >= A.B * Hk) return;
            stride = WARPS;
            at.b = blockIdx.x / Hk, at.h = blockIdx.x - at.b * Hk, at.ubeg = 0;
            x0 = warp, x1 = 1 << 30;
        } else {
            int before = scan - mine, all = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                before += w < warp ? s_scan[w] : 0;
                all += s_scan[w];
            }
            all *= Hk;
            chunk = (all + workers - 1) / workers;
            int off = before * Hk;
            for (int b = b0; b < b1; ++b) {
                const int v = places(tokens_of(A.lens, b, A.blocks)) * Hk;
#pragma unroll 1
                for (int w = 0; w < WARPS; ++w) {
                    const i64 x = (i64)(w * gridDim.x + blockIdx.x) * chunk;
                    if (x >= off && x < off + v) s_scan[WARPS + 2 * w] = b, s_scan[WARPS + 2 * w + 1] = off;
                }
                off += v;
            }
            __syncthreads();
            if ((i64)me * chunk >= all) return;
            x0 = me * chunk, x1 = min(x0 + chunk, all);
            at.b = s_scan[WARPS + 2 * warp];
            const int vp = places(tokens_of(A.lens, at.b, A.blocks));
            at.h = (x0 - s_scan[WARPS + 2 * warp + 1]) / vp;
            at.ubeg = s_scan[WARPS + 2 * warp + 1] + at.h * vp;
        }
    }
    auto measure = [&](Place& p) {
        const int len = tokens_of(A.lens, p.b, A.blocks);
        p.np = (len + kBlk - 1) / kBlk;
        p.vp = max(1, p.np);
    };
    measure(at);
    if (whole) at.ubeg = 0;
    if (whole || stride > 1) x1 = at.vp;
    // The next unit of the range; false at its end.
    auto next_unit = [&](Place& p, int& end) -> bool {
        if (whole) {
            const int u = p.b * Hk + p.h + workers;
            if (u >= A.B * Hk) return false;
            p.b = u / Hk, p.h = u - p.b * Hk;
            measure(p);
            p.ubeg = 0, end = p.vp;
            return true;
        }
        p.ubeg += p.vp;
        if (p.ubeg >= end) return false;
        if (++p.h == Hk) {
            p.h = 0;
            ++p.b;
            measure(p);
        }
        return true;
    };

    // ---- the producer: half pages of this warp's pages, in order, NH - 1 ahead of their use
    Place pat = at;
    int px = x0, pend = x1, pid = 0, pslot = 0;
    bool pmore = true;
    auto p_settle = [&]() {                      // move px to the warp's next place that is a page
        for (;;) {
            if (px >= min(pat.ubeg + pat.vp, pend)) {
                if (!next_unit(pat, pend)) {
                    pmore = false;
                    return;
                }
                if (whole) px = 0;
                continue;
            }
            if (px - pat.ubeg < pat.np) break;
            px += stride;
        }
        pid = page_of(A.table + (i64)pat.b * A.blocks, px - pat.ubeg, A.cache.pages);
    };
    p_settle();
    bool p_values = false;
    auto issue = [&]() {
        if (pmore) {
            const i64 ph = (i64)pid * Hk + pat.h;
            const char* src = reinterpret_cast<const char*>(p_values ? A.cache.v : A.cache.k) + ph * P::HALF;
            char* dst = ring + pslot * P::HALF;
            if (!p_values) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const int c = lane + 32 * i, r = c / (D / 16), cc = c - r * (D / 16);
                    cp_async16(dst + (r * (D / 16) + key_chunk<D>(r, cc)) * 16, src + c * 16);
                }
                if (lane < 2) {
                    const float* s = (lane ? A.cache.v_scale : A.cache.k_scale) + ph;
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((u32)__cvta_generic_to_shared(
                                     reinterpret_cast<float*>(hdr + pslot) + lane)), "l"(s) : "memory");
                }
            } else {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) cp_async16(dst + (lane + 32 * i) * 16, src + (lane + 32 * i) * 16);
                px += stride;
                p_settle();
            }
            p_values = !p_values;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        pslot = pslot + 1 == NH ? 0 : pslot + 1;
    };
#pragma unroll 1
    for (int i = 0; i < NH - 1; ++i) issue();
    int slot = 0;
    auto take = [&]() -> const char* {            // the next half page, complete; requests the one NH - 1 behind it
        asm volatile("cp.async.wait_group %0;" ::"n"(NH - 2) : "memory");
        __syncwarp();
        const char* p = ring + slot * P::HALF;
        issue();
        return p;
    };

    // ---- the consumer
    int end = x1;
    int x = x0;
    for (;;) {
        const int len = tokens_of(A.lens, at.b, A.blocks), cnt = queries_of(A.count, at.b, A.T);
        // query rows r = t * group + g of this head, as FP16 columns scaled by a power of two; a lane loads row 8 nt + n and
        // keeps the scores of rows 8 nt + 2 t + e
        u32 qb[NT][KS][2];
        float crow[NT][2];
        int limit[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = 8 * nt + n, tq = (int)fdiv((unsigned)r, A.by_group);
            const bool live = r < R && tq < cnt;
            const u16* qr = A.q + at.b * A.q_sb + tq * A.q_st + (i64)(at.h * A.group + r - tq * A.group) * D;
            float v[KS][4], amax = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                // the four elements that lane t contributes to step s (see the key loads)
                const int d = s < D / 64 * 4 ? 64 * (s / 4) + 16 * t + 4 * (s % 4)
                            : s < D / 32 * 2 ? D / 64 * 64 + 8 * t + 4 * (s - D / 64 * 4) : D / 32 * 32 + 4 * t;
                const uint2 w = live ? *reinterpret_cast<const uint2*>(qr + d) : make_uint2(0u, 0u);
                unpack2<DT>(w.x, v[s][0], v[s][1]);
                unpack2<DT>(w.y, v[s][2], v[s][3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(v[s][e]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            float back;
            const float up = row_scale(amax, back);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qb[nt][s][0] = half2_of(v[s][0] * up, v[s][1] * up);
                qb[nt][s][1] = half2_of(v[s][2] * up, v[s][3] * up);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int rs = 8 * nt + 2 * t + e, ts = (int)fdiv((unsigned)rs, A.by_group);
                crow[nt][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + e)) * A.scale_log2;
                limit[nt][e] = rs >= R || ts >= cnt ? 0 : A.causal ? min(max(len - cnt + ts + 1, 0), len) : len;
            }
        }
        const int open = A.causal ? len - cnt + 1 : len;         // keys below this are seen by every query
        float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }
        const int seg_end = min(at.ubeg + at.vp, end);
#pragma unroll 1
        for (; x < seg_end; x += stride) {
            const int pg = x - at.ubeg;
            if (pg >= at.np) continue;
            const float2* sp = hdr + slot;
            const char* kp = take();
            const float2 sc = *sp;
            slot = slot + 1 == NH ? 0 : slot + 1;
            // scores: tile j holds blocks 2 j (rows 0..7) and 2 j + 1
            float s[NT][4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 16 * (n >> 1) + 4 * j + (n & 1);
                const char *ra = kp + r * D, *rb = ra + 2 * D;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][j][0] = s[nt][j][1] = s[nt][j][2] = s[nt][j][3] = 0.f;
                auto step = [&](int ks, u32 wa, u32 wb) {
                    u32 a0, a1, a2, a3;
                    int8x4_to_half(wa, a0, a2);
                    int8x4_to_half(wb, a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(s[nt][j], a0, a1, a2, a3, qb[nt][ks][0], qb[nt][ks][1]);
                };
#pragma unroll
                for (int q4 = 0; q4 < D / 64; ++q4) {
                    const uint4 u = *reinterpret_cast<const uint4*>(ra + key_chunk<D>(r, 4 * q4 + t) * 16);
                    const uint4 v = *reinterpret_cast<const uint4*>(rb + key_chunk<D>(r + 2, 4 * q4 + t) * 16);
                    step(4 * q4, u.x, v.x), step(4 * q4 + 1, u.y, v.y), step(4 * q4 + 2, u.z, v.z), step(4 * q4 + 3, u.w, v.w);
                }
                if (D % 64 >= 32) {
                    const uint2 u = *reinterpret_cast<const uint2*>(ra + D / 64 * 64 + 8 * t), v = *reinterpret_cast<const uint2*>(rb + D / 64 * 64 + 8 * t);
                    step(D / 64 * 4, u.x, v.x), step(D / 64 * 4 + 1, u.y, v.y);
                }
                if (D % 32)
                    step(D / 32 * 2, *reinterpret_cast<const u32*>(ra + D / 32 * 32 + 4 * t), *reinterpret_cast<const u32*>(rb + D / 32 * 32 + 4 * t));
            }
            const float vs = safe_scale(sc.y), bias = lg2(vs), inv = rcp(vs);
            const bool masked = (pg + 1) * kBlk > open;
            u32 pb[NT][4][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float top[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float c = crow[nt][e] * sc.x;
                    if (masked) {
                        const int lim = limit[nt][e] - pg * kBlk - 16 * (n >> 1) - (n & 1);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            s[nt][j][e] = 4 * j < lim ? __fmaf_rn(s[nt][j][e], c, bias) : -INFINITY;
                            s[nt][j][2 + e] = 4 * j + 2 < lim ? __fmaf_rn(s[nt][j][2 + e], c, bias) : -INFINITY;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            s[nt][j][e] = __fmaf_rn(s[nt][j][e], c, bias);
                            s[nt][j][2 + e] = __fmaf_rn(s[nt][j][2 + e], c, bias);
                        }
                    }
                    top[e] = fmaxf(fmaxf(fmaxf(s[nt][0][e], s[nt][0][2 + e]), fmaxf(s[nt][1][e], s[nt][1][2 + e])),
                                   fmaxf(fmaxf(s[nt][2][e], s[nt][2][2 + e]), fmaxf(s[nt][3][e], s[nt][3][2 + e])));
                }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
                }
                const bool move0 = top[0] > m[nt][0] + kSlack, move1 = top[1] > m[nt][1] + kSlack;
                if (__any_sync(0xffffffffu, move0 || move1)) {
                    const float f0 = move0 ? ex2(m[nt][0] - top[0]) : 1.f, f1 = move1 ? ex2(m[nt][1] - top[1]) : 1.f;
                    if (move0) m[nt][0] = top[0];
                    if (move1) m[nt][1] = top[1];
                    l[nt][0] *= f0, l[nt][1] *= f1;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) o[nt][i][0] *= f0, o[nt][i][1] *= f1, o[nt][i][2] *= f0, o[nt][i][3] *= f1;
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float base = (m[nt][e] == -INFINITY ? 0.f : m[nt][e]) - kRef;
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[nt][j][e] = ex2(s[nt][j][e] - base), s[nt][j][2 + e] = ex2(s[nt][j][2 + e] - base);
                        sum += s[nt][j][e] + s[nt][j][2 + e];
                    }
                    l[nt][e] = __fmaf_rn(sum, inv, l[nt][e]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    pb[nt][j][0] = turned(half2_of(s[nt][j][0], s[nt][j][1]));
                    pb[nt][j][1] = turned(half2_of(s[nt][j][2], s[nt][j][3]));
                }
            }
            if (sc.y < kLeastScale) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) pb[nt][j][0] = pb[nt][j][1] = 0u;
            }
            const char* vp = take();
            slot = slot + 1 == NH ? 0 : slot + 1;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const uint4 u = *reinterpret_cast<const uint4*>(vp + (16 * i + n) * kBlk + 16 * t);
                const uint4 v = *reinterpret_cast<const uint4*>(vp + (16 * i + 8 + n) * kBlk + 16 * t);
                const u32 uu[4] = {u.x, u.y, u.z, u.w}, vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u32 a0, a1, a2, a3;
                    int8x4_to_half(uu[j], a0, a2);
                    int8x4_to_half(vv[j], a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][i], a0, a1, a2, a3, pb[nt][j][0], pb[nt][j][1]);
                }
            }
        }
        // ---- the unit's rows, or this worker's part of them
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float& v = l[nt][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
                if (limit[nt][e] == 0) v = 0.f;               // a row that sees no token
            }
        auto out_row = [&](int r) -> u16* {
            const int tq = (int)fdiv((unsigned)r, A.by_group);
            return A.out + (((i64)at.b * A.T + tq) * A.heads + at.h * A.group + r - tq * A.group) * D;
        };
        // a part: rows of D sums, the reference and the sum of weights
        auto write_part = [&](float* part) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * nt + 2 * t + e;
                    if (r >= R) continue;
                    float* row = part + r * (D + 2);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) row[16 * i + n] = o[nt][i][e], row[16 * i + 8 + n] = o[nt][i][2 + e];
                    if (n == 0) row[D] = m[nt][e], row[D + 1] = l[nt][e];
                }
        };
        if (stride > 1) {
            __syncwarp();
            write_part(reinterpret_cast<float*>(ring));
            __syncthreads();
            for (int i = tid; i < R * (D / 2); i += WARPS * 32) {
                const int r = i / (D / 2), d = 2 * (i - r * (D / 2));
                const char* part = smem + r * (D + 2) * 4;
                float top = -INFINITY, sum = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) top = fmaxf(top, reinterpret_cast<const float*>(part + w * NH * P::HALF)[D]);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    const float* row = reinterpret_cast<const float*>(part + w * NH * P::HALF);
                    const float f = top == -INFINITY ? 0.f : ex2(row[D] - top);
                    sum = __fmaf_rn(row[D + 1], f, sum), a0 = __fmaf_rn(row[d], f, a0), a1 = __fmaf_rn(row[d + 1], f, a1);
                }
                const float f = sum != 0.f ? 1.f / sum : 0.f;
                *reinterpret_cast<u32*>(out_row(r) + d) = pack2<DT>(a0 * f, a1 * f);
            }
            break;
        }
        if (at.ubeg >= (whole ? 0 : x0) && seg_end == at.ubeg + at.vp) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float f0 = l[nt][0] != 0.f ? 1.f / l[nt][0] : 0.f, f1 = l[nt][1] != 0.f ? 1.f / l[nt][1] : 0.f;
                const int r = 8 * nt + n;                     // after the turn a lane holds row n, elements 2 t and 2 t + 1
                u32* dst = reinterpret_cast<u32*>(out_row(r));
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const u32 lo = turned(pack2<DT>(o[nt][i][0] * f0, o[nt][i][1] * f1)), hi = turned(pack2<DT>(o[nt][i][2] * f0, o[nt][i][3] * f1));
                    if (r < R) dst[8 * i + t] = lo, dst[8 * i + 4 + t] = hi;
                }
            }
        } else {
            // More than 16 parts are added in two steps, sixteen neighbours first (one warp over 222 parts of one token and
            // 131037 keys took as long as the pages: 84 -> 47 us).
            const int first = at.ubeg / chunk, last = (at.ubeg + at.vp - 1) / chunk;
            constexpr i64 SIZE = (i64)(8 * NT) * (D + 2);
            write_part(A.part + part_slot(me, first) * SIZE);
            // true in the warp that arrives last
            auto arrive = [&](int* counter, int expected) -> bool {
                __threadfence();
                __syncwarp();
                int seen = 0;
                if (lane == 0) seen = atomicAdd(counter, 1);
                seen = __shfl_sync(0xffffffffu, seen, 0);
                if (seen != expected - 1) return false;
                if (lane == 0) *counter = 0;
                __threadfence();
                return true;
            };
            int step = 1;
            bool add = true;
            if (last - first >= 16) {
                const int lead = first + (me - first) / 16 * 16, end16 = min(lead + 15, last);
                add = arrive(A.counters + workers + part_slot(lead, first), end16 - lead + 1);
                if (add) add_parts<DT, D>(A.part, SIZE, first, lead, end16, 1, R, A.group, nullptr, 0);
                step = 16;
            }
            if (add && arrive(A.counters + first, (last - first) / step + 1))
                add_parts<DT, D>(A.part, SIZE, first, first, last, step, R, A.group, out_row(0), (i64)A.heads * D);
        }
        if (!next_unit(at, end)) break;
        if (whole) x = 0;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// ------------------------------------------------------------------------------------------------ many query rows
// Frames and prompts: tensor-core products (tcgen05) on tiles of 128 query rows and 128 keys (two pages).
//
// The rows of a key head are its queries in token order, `group` heads to a token, so a causal limit never falls along the
// rows. A CTA takes NG groups of up to 128 rows and one key head. Roles:
//   softmax   256 threads per group, two to a row, a page of the tile each: 64 scores from TMEM, weights (FP16) back to TMEM
//             over the scores. The two agree on the row's reference at a named barrier before either writes;
//   product   one warp, an elected lane of which issues S = Q K^T (both operands in shared memory) and O += P V (P in TMEM);
//   convert   what is left: INT8 pages, copied asynchronously a tile ahead, to FP16 tiles in shared memory, 128-byte swizzled,
//             keys K-major along the head, values K-major along the tokens.
// The two groups alternate: while one's weights are formed, the other's products run. Mathematics, scaling of the queries and
// handling of the scales are those of the few-row kernel; the reference m moves only when a score passes it by 10.5, and O (in
// TMEM) is rescaled by its own row's threads. S of a tile is issued after O of the tile before it, and a commit covers every
// product issued before it: scores that have arrived mean that O is complete up to the tile before.
//
// Bound by the softmax warps' chain per tile (about 3,700 clocks at head width 64, 4,000 at 128: scores 500 .. 900, load 200,
// maximum and barrier 500, weights 1,400 .. 1,950, of which the exponential unit alone needs 2,048 for both groups, handing over
// and the loop 700), not by the products (1,024 and 2,048 clocks): 2 x 4096 queries of 32 heads of 128, 8 key heads, 4200 keys: 345 to
// 351 us, 823 to 838 TFLOP/s; 160 queries over 16411 keys, heads of 64: 60.5 us. Measured on the way to this shape, same two cases: one thread to a row with two
// passes over the scores 423 and 73 us; products issued from a single-lane branch (130 clocks each instead of 64) 448 and 74;
// a row per lane for loads and stores of Q and O 376 and 67 us; scores a tile ahead in TMEM columns of their own (heads up to 64)
// 64 us at the second; an eighth to a third of the exponentials by polynomial: no faster.
//
// Few units (a frame of one robot): the tiles of a unit are divided over a cluster of CTAs, which add their parts through
// distributed shared memory. Into how many goes by the table's width, the host's bound on the lengths: a table of another
// width may add the parts in another order.

constexpr int kTile = 128;            // keys of a tile, rows of a group

template <int D, int NG>
struct Many {
    static constexpr int ATOMS = (D + 63) / 64;                       // 64-element columns of a K-major tile
    static constexpr int QB = kTile * 128 * ATOMS;                    // bytes of a group's queries
    static constexpr int KB = kTile * 128 * ATOMS;                    // of a tile's keys
    static constexpr int VB = D * 128 * 2;                            // of its values
    static constexpr int NS = 2;                                      // tiles of either in flight
    // Threads and registers. With two groups the CTA is launched with 80 registers a thread (768 x 80), of which the softmax
    // warps take more and the others less: 512 x 96 + 256 x 48 = 61,440 (launch_many checks the 80).
    static constexpr int LAUNCH_REGS = 80;
    static constexpr int SOFT = NG * 256;                            // softmax threads: two to a row, a page each
    static constexpr int THREADS = NG == 2 ? 768 : 512;
    static constexpr int CONV = THREADS - SOFT - 32;                 // convert threads: what softmax and the product warp leave
    static constexpr int PAGE = kBlk * D;                             // bytes of a page's keys or values
    static constexpr int RING = 4;                                    // INT8 pages on their way (a tile's keys and values)
    static constexpr int Q0 = 0, K0 = NG * QB, V0 = K0 + NS * KB, STAGE0 = V0 + NS * VB, BAR0 = STAGE0 + RING * PAGE;
    static constexpr int SWAP0 = BAR0 + 256;                          // a float of every softmax thread
    static constexpr int BYTES = SWAP0 + SOFT * 4;
    static constexpr int ML0 = STAGE0;                                // m, l of every row, over the stage (cluster sums)
    static constexpr u32 COLS = NG == 2 ? 512 : 256;
    static constexpr int S0 = 0, O0 = NG * kTile;                     // TMEM columns: scores, outputs
    static constexpr int PARTS = NG * kTile * D * 4;                  // a CTA's part of the outputs, over the tiles
    static_assert(PARTS <= STAGE0 && NG * kTile * 8 <= RING * PAGE, "the parts overlay the tiles, their sums the stage");
};

// 16 bytes to shared memory, zeros when !there.
__device__ __forceinline__ void cp_async16_zfill(u32 dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// The barriers of a CTA, 8 bytes each from BAR0.
enum { BAR_KFULL = 0, BAR_KEMPTY = 2, BAR_VFULL = 4, BAR_VEMPTY = 6, BAR_SFULL = 8, BAR_PFULL = 10, BAR_Q = 14, BAR_O = 15, BAR_COUNT = 16 };

template <int DT, int D, int NG>
__global__ void __launch_bounds__(Many<D, NG>::THREADS, 1)
k_attention_many(const AttnArgs A, int row_tiles, int tile_rows, int splits) {
    typedef Many<D, NG> P;
    constexpr int KS = D / 16, NC = (8 * D + P::CONV - 1) / P::CONV;      // contraction steps; 16-byte chunks of half a tile per convert thread
    extern __shared__ __align__(1024) char smem_tiles[];
    char* const smem = smem_tiles;
    const u32 sbase = smem_u32(smem), bars = sbase + P::BAR0;
    u32* tmem_slot = reinterpret_cast<u32*>(smem + P::BAR0 + 8 * BAR_COUNT);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    constexpr int W_MMA = NG * 8, W_CONV = W_MMA + 1;
    auto bar = [&](int i) -> u32 { return bars + 8 * i; };
    auto wait = [&](int i, u32 parity) -> bool { return mbar_wait_suspended(bar(i), parity & 1, abort_flag, &g_tcq_attention_error); };
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(BAR_KFULL + i), P::CONV / 32);    // one arrival per convert warp
            mbar_init(bar(BAR_VFULL + i), P::CONV / 32);
            mbar_init(bar(BAR_KEMPTY + i), 1);
            mbar_init(bar(BAR_VEMPTY + i), 1);
            mbar_init(bar(BAR_SFULL + i), 1);
            mbar_init(bar(BAR_PFULL + i), 4);               // per softmax warp; group and page at 2 g + p
            mbar_init(bar(BAR_PFULL + 2 + i), 4);
        }
        mbar_init(bar(BAR_Q), P::SOFT);
        mbar_init(bar(BAR_O), 1);
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

    // ---- the unit: rows r0 .. r0 + tile_rows - 1 of key head h of sequence b (the heaviest row tiles of causal launches
    // first), and this CTA's tiles [k0, k1) of its keys
    const int Hk = A.cache.kv_heads, R = A.T * A.group;
    const int sp = blockIdx.x % splits, unit = blockIdx.x / splits, bh = unit % (A.B * Hk), b = bh / Hk, h = bh - b * Hk;
    const int rt = row_tiles - 1 - unit / (A.B * Hk), r0 = rt * tile_rows, r1 = min(R, r0 + tile_rows);
    const int len = tokens_of(A.lens, b, A.blocks), cnt = queries_of(A.count, b, A.T);
    const int last_q = min((int)fdiv((unsigned)(r1 - 1), A.by_group), cnt - 1), first_q = (int)fdiv((unsigned)r0, A.by_group);
    const int upto = last_q < first_q ? 0 : A.causal ? min(max(len - cnt + last_q + 1, 0), len) : len;     // keys that some row sees
    const int open = A.causal ? len - cnt + first_q + 1 : len;                                             // and that every row sees
    const int tiles = (upto + kTile - 1) / kTile;
    const int k0 = (int)((i64)tiles * sp / splits), k1 = (int)((i64)tiles * (sp + 1) / splits);
    const int pages = (upto + kBlk - 1) / kBlk;
    const int* trow = A.table + (i64)b * A.blocks;

    float m = -INFINITY, l = 0.f;
    if (NG == 2) {
        if (warp < W_MMA) asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    }
    if (warp < W_MMA) {
        // ------------------------------------------------------------------------------------------------ softmax
        const int g = warp >> 3, p = (warp >> 2) & 1, gl = tid & 127, r = r0 + g * kTile + gl, tq = (int)fdiv((unsigned)r, A.by_group);
        const int pair_bar = 1 + g * 4 + (warp & 3);            // the two warps of 32 rows meet at a named barrier
        const bool live = r < r1 && tq < cnt;
        const int limit = !live ? 0 : A.causal ? min(max(len - cnt + tq + 1, 0), len) : len;
        float crow = 0.f;
        float* swap = reinterpret_cast<float*>(smem + P::SWAP0);
        const int mine = (g * 2 + p) * kTile + gl, other = mine ^ kTile;
        if (k1 > k0) {
            // Queries to shared memory: SEG lanes to a row (16 bytes each), a warp's 16 rows requested at once; each row scaled
            // by a power of two, which its own threads then take from the swap area.
            constexpr int LPR = D / 8, SEG = LPR <= 4 ? 4 : LPR <= 8 ? 8 : 16, RPP = 32 / SEG, NP = 16 / RPP;
            const int sl = lane % SEG, w8 = warp & 7;
            uint4 w[NP];
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const int row = w8 * 16 + n * RPP + lane / SEG, rr = r0 + g * kTile + row, tt = (int)fdiv((unsigned)rr, A.by_group);
                const u16* qr = A.q + b * A.q_sb + tt * A.q_st + (i64)(h * A.group + rr - tt * A.group) * D;
                w[n] = rr < r1 && tt < cnt && sl < LPR ? reinterpret_cast<const uint4*>(qr)[sl] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const int row = w8 * 16 + n * RPP + lane / SEG;
                u32 ww[4] = {w[n].x, w[n].y, w[n].z, w[n].w};
                float amax = 0.f, x, y;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unpack2<DT>(ww[j], x, y);
                    amax = max3(amax, fabsf(x), fabsf(y));
                }
#pragma unroll
                for (int o = 1; o < SEG; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                float back, up = row_scale(amax, back);
                if (A.scale_log2 < 0.f) up = -up;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unpack2<DT>(ww[j], x, y);
                    ww[j] = half2_of(x * up, y * up);
                }
                if (sl < LPR)
                    *reinterpret_cast<uint4*>(smem + P::Q0 + g * P::QB + (sl >> 3) * (kTile * 128) + row * 128 + (((sl & 7) ^ (row & 7)) << 4)) =
                        make_uint4(ww[0], ww[1], ww[2], ww[3]);
                if (sl == 0) swap[g * 2 * kTile + row] = back;
            }
            async_proxy_fence();
            asm volatile("barrier.cta.sync 15, %0;" ::"r"(P::SOFT) : "memory");
            mbar_arrive(bar(BAR_Q));
            crow = swap[g * 2 * kTile + gl] * fabsf(A.scale_log2);
            pair_sync(pair_bar);                              // both have read it before either swaps
        }
        const u32 lanes = (u32)((warp & 3) * 32) << 16, ts = tmem + lanes + P::S0 + g * kTile, to = tmem + lanes + P::O0 + g * D;
        // the scales of this thread's page of the next tile are requested a tile ahead, the page's number two
        int id = 0;
        float nk = 0.f, nv = 1.f;
        auto request_id = [&](int i) {
            if (i < k1) id = trow[min(2 * i + p, pages - 1)];
        };
        auto request_scales = [&](int i) {
            if (i < k1) {
                const i64 ph = (i64)page_in(id, A.cache.pages) * Hk + h;
                nk = A.cache.k_scale[ph], nv = A.cache.v_scale[ph];
            }
        };
        request_id(k0);
        request_scales(k0);
        request_id(k0 + 1);
        // One page of a tile: its 64 scores into registers, their largest, weights back over the scores. The pair agrees on the
        // row's reference before either writes a weight: nothing of S is read after that, and no product reads or adds to the
        // rows before both pages' weights have been handed over. Returns false when a wait expired.
        auto tile = [&](auto masked_c, int i, float c, float vsc) -> bool {
            constexpr bool MASKED = decltype(masked_c)::value;
            const float vs = safe_scale(vsc), bias = lg2(vs), inv = rcp(vs);
            const int lim = limit - i * kTile - 64 * p;
            const bool ok = wait(BAR_SFULL + g, i - k0);
            tc_after();
            u32 v[2][32];
            tmem_ld32(ts + 64 * p, v[0]);
            tmem_ld32(ts + 64 * p + 32, v[1]);
            tmem_ld_wait(v[0]);
            tmem_ld_wait(v[1]);
            float raw[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 64; j += 2) {
                float x = __uint_as_float(v[j >> 5][j & 31]), y = __uint_as_float(v[j >> 5][(j & 31) + 1]);
                if (MASKED) {
                    x = j < lim ? x : -INFINITY;
                    y = j + 1 < lim ? y : -INFINITY;
                }
                raw[(j >> 1) & 3] = max3(raw[(j >> 1) & 3], x, y);
            }
            float top = fmaxf(fmaxf(raw[0], raw[1]), fmaxf(raw[2], raw[3]));
            if (!MASKED || top != -INFINITY) top = __fmaf_rn(top, c, bias);
            // The pair's barrier stands between this warp's loads of the scores and the other's weights over the same columns:
            // with a fence on either side it orders them.
            tc_before();
            const bool moves = pair_any(pair_bar, top > m + kSlack || !ok);
            tc_after();
            if (moves) {
                // Move the reference up where a score passed it: O and the sum follow. An expired wait is told as a NaN that no
                // arithmetic makes, so that both warps leave.
                constexpr u32 gone = 0x7fffdeadu;
                swap[mine] = ok ? top : __uint_as_float(gone);
                pair_sync(pair_bar);
                const float theirs = swap[other], both = fmaxf(top, theirs);
                if (__any_sync(0xffffffffu, !ok || __float_as_uint(theirs) == gone)) return false;
                const bool move = both > m + kSlack;
                const float f = move ? ex2(m - both) : 1.f;
                if (move) m = both;
                l *= f;
                if (i > k0) {
#pragma unroll 1
                    for (int d = p * (D / 2); d < (p + 1) * (D / 2); d += 8) {
                        u32 o[8];
                        tmem_ld8(to + d, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                        tmem_st8(to + d, o);
                    }
                    tmem_st_wait();
                    tc_before();
                }
                pair_sync(pair_bar);
                tc_after();
            }
            const float base = (m == -INFINITY ? 0.f : m) - kRef;
            const u64 c2 = pair(c, c), a2 = pair(bias - base, bias - base);
            u64 sum[2] = {0, 0};
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                u32(&x)[32] = v[hf];
                u32 w[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const u64 y = fma2(pair(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), c2, a2);
                    float lo, hi;
                    unpair(y, lo, hi);
                    if (MASKED) {
                        lo = 32 * hf + 2 * j < lim ? lo : -INFINITY;
                        hi = 32 * hf + 2 * j + 1 < lim ? hi : -INFINITY;
                    }
                    lo = ex2(lo), hi = ex2(hi);
                    sum[j & 1] = add2(sum[j & 1], pair(lo, hi));
                    w[j] = half2_of(lo, hi);
                }
                tmem_st16(ts + 32 * p + 16 * hf, w);
            }
            float lo, hi;
            unpair(add2(sum[0], sum[1]), lo, hi);
            l = __fmaf_rn(lo + hi, inv, l);
            tmem_st_wait();
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(BAR_PFULL + 2 * g + p));
            return true;
        };
        // Warps without a query (the last rows of a tile, sequences with fewer queries) only keep the barriers going: what their
        // TMEM lanes hold stays in their own rows.
        const bool idle = !__any_sync(0xffffffffu, live);
#pragma unroll 1
        for (int i = k0; i < k1; ++i) {
            if (idle) {
                if (!wait(BAR_SFULL + g, i - k0)) break;
                if (lane == 0) mbar_arrive(bar(BAR_PFULL + 2 * g + p));
                continue;
            }
            const float c = crow * nk, vsc = nv;
            request_scales(i + 1);
            request_id(i + 2);
            if (!((i + 1) * kTile > open ? tile(std::true_type(), i, c, vsc) : tile(std::false_type(), i, c, vsc))) break;
        }
        // the row's sum from its two threads, its elements half by half
        swap[mine] = limit == 0 ? 0.f : l;
        pair_sync(pair_bar);
        l = swap[mine & ~kTile] + swap[mine | kTile];
        const bool got = k1 > k0 && wait(BAR_O, 0);
        tc_after();
        // Rows to shared memory, over the tiles (every product is done), 16-byte chunks permuted within a row: FP32 parts for
        // the cluster's sum, or the output's values for stores of whole rows.
        const float f = splits > 1 ? 1.f : l != 0.f ? 1.f / l : 0.f;
        const int row = g * kTile + gl;
#pragma unroll 1
        for (int d = p * (D / 2); d < (p + 1) * (D / 2); d += 8) {
            u32 o[8] = {};
            if (got) {
                tmem_ld8(to + d, o);
                tmem_ld_wait(o);
            }
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = l != 0.f ? __uint_as_float(o[j]) * f : 0.f;
            if (splits > 1) {
                constexpr int X = (D / 4) % 8 == 0 ? 7 : 3;
                float4* part = reinterpret_cast<float4*>(smem) + row * (D / 4);
                part[(d / 4) ^ (row & X)] = make_float4(y[0], y[1], y[2], y[3]);
                part[(d / 4 + 1) ^ (row & X)] = make_float4(y[4], y[5], y[6], y[7]);
            } else {
                constexpr int X = (D / 8) % 8 == 0 ? 7 : (D / 8) % 4 == 0 ? 3 : 1;
                reinterpret_cast<uint4*>(smem)[row * (D / 8) + ((d / 8) ^ (row & X))] =
                    make_uint4(pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]), pack2<DT>(y[4], y[5]), pack2<DT>(y[6], y[7]));
            }
        }
        if (splits > 1) {
            if (p == 0) reinterpret_cast<float2*>(smem + P::ML0)[row] = make_float2(got ? m : -INFINITY, got ? l : 0.f);
        } else {
            constexpr int X = (D / 8) % 8 == 0 ? 7 : (D / 8) % 4 == 0 ? 3 : 1;
            asm volatile("barrier.cta.sync 15, %0;" ::"r"(P::SOFT) : "memory");
            for (int e = tid; e < (r1 - r0) * (D / 8); e += P::SOFT) {
                const int rr = e / (D / 8), ch = e - rr * (D / 8), t = (int)fdiv((unsigned)(r0 + rr), A.by_group);
                u16* dst = A.out + (((i64)b * A.T + t) * A.heads + h * A.group + r0 + rr - t * A.group) * D;
                reinterpret_cast<uint4*>(dst)[ch] = reinterpret_cast<const uint4*>(smem)[rr * (D / 8) + (ch ^ (rr & X))];
            }
        }
    } else if (warp >= W_CONV) {
        // ------------------------------------------------------------------------------------------------ convert
        // Halves of a tile: its two pages' keys, its two pages' values. A half's INT8 data is requested a tile ahead of its use
        // (asynchronous copies of each thread's own 16-byte chunks), the pages' numbers two tiles.
        const int ct = tid - W_CONV * 32;
        int id[2] = {}, koff[NC], voff[NC];
        float least[2] = {1.f, 1.f};                     // value scales of the tile last requested
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            // where chunk c of a half (16 elements) goes: 32 bytes of a key's row, of a value's row
            const int c = ct + P::CONV * n, p = c >= 4 * D, cc = c - p * 4 * D, kr = cc / (D / 16), kx = cc - kr * (D / 16), vr = cc >> 2, vx = cc & 3;
            koff[n] = P::K0 + (kx >> 2) * (kTile * 128) + (64 * p + kr) * 128 + (((2 * (kx & 3)) ^ (kr & 7)) << 4);
            voff[n] = P::V0 + (p * D + vr) * 128 + (((2 * vx) ^ (vr & 7)) << 4);
        }
        auto request_ids = [&](int i) {
            if (i < k1) id[0] = trow[2 * i], id[1] = trow[min(2 * i + 1, pages - 1)];
        };
        auto request = [&](int i, int vals) {
            if (i < k1) {
                const bool two = 2 * i + 1 < pages;
                const i64 p0 = (i64)page_in(id[0], A.cache.pages) * Hk + h, p1 = (i64)page_in(id[1], A.cache.pages) * Hk + h;
                const i8* cells = vals ? A.cache.v : A.cache.k;
                const i8 *s0 = cells + p0 * P::PAGE, *s1 = cells + (p1 - 1) * P::PAGE;
                if (vals) least[0] = A.cache.v_scale[p0], least[1] = A.cache.v_scale[p1];
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    const int c = ct + P::CONV * n;
                    const bool p = c >= 4 * D;
                    if (NC * P::CONV == 8 * D || c < 8 * D)
                        cp_async16_zfill(sbase + P::STAGE0 + vals * 2 * P::PAGE + c * 16, (p ? s1 : s0) + c * 16, two || !p);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        request_ids(k0);
        request(k0, 0);
        request(k0, 1);
        request_ids(k0 + 1);
#pragma unroll 1
        for (int i = k0; i < k1; ++i) {
            const int it = i - k0, s = it & 1, use = it >> 1;
            bool ok = true;
#pragma unroll 1
            for (int vals = 0; vals < 2; ++vals) {
                ok = wait((vals ? BAR_VEMPTY : BAR_KEMPTY) + s, use + 1);
                if (!ok) break;
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                const int dst = s * (vals ? P::VB : P::KB);
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    const int c = ct + P::CONV * n;
                    if (NC * P::CONV != 8 * D && c >= 8 * D) break;
                    uint4 q = *reinterpret_cast<const uint4*>(smem + P::STAGE0 + vals * 2 * P::PAGE + c * 16);
                    if (vals && (c >= 4 * D ? least[1] : least[0]) < kLeastScale) q = make_uint4(0, 0, 0, 0);     // values that count as zero
                    u32 w[8];
                    int8x4_to_half(q.x, w[0], w[1]);
                    int8x4_to_half(q.y, w[2], w[3]);
                    int8x4_to_half(q.z, w[4], w[5]);
                    int8x4_to_half(q.w, w[6], w[7]);
                    const int o = (vals ? voff[n] : koff[n]) + dst;
                    *reinterpret_cast<uint4*>(smem + o) = make_uint4(w[0], w[1], w[2], w[3]);
                    *reinterpret_cast<uint4*>(smem + (o ^ 16)) = make_uint4(w[4], w[5], w[6], w[7]);
                }
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar((vals ? BAR_VFULL : BAR_KFULL) + s));
                request(i + 1, vals);
            }
            if (!ok) break;
            request_ids(i + 2);
        }
        cp_async_wait_all();
    } else if (k1 > k0) {
        // ------------------------------------------------------------------------------------------------ product
        // The whole warp runs this loop, so that descriptors and addresses stay in uniform registers; one elected lane
        // issues (issued from a single-lane branch, each product took about 130 clocks instead of the 64 of its arithmetic).
        const u64 qd = sw128_desc(sbase + P::Q0), kd = sw128_desc(sbase + P::K0), vd = sw128_desc(sbase + P::V0);
        auto scores = [&](int g, int s) {
            if (elect_one()) {
                const u64 a = qd + (u32)(g * (P::QB >> 4)), b = kd + (u32)(s * (P::KB >> 4));
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    constexpr u32 atom = kTile * 128 / 16;
                    mma_ss(tmem + P::S0 + g * kTile, a + ((k >> 2) * atom + 2 * (k & 3)), b + ((k >> 2) * atom + 2 * (k & 3)), idesc_f16(kTile), k > 0);
                }
                mma_commit(bar(BAR_SFULL + g));
            }
            __syncwarp();
        };
        auto commit = [&](int i) {
            if (elect_one()) mma_commit(bar(i));
            __syncwarp();
        };
        const int n = k1 - k0;
        bool ok = wait(BAR_Q, 0) && wait(BAR_KFULL, 0);
        if (ok) {
            tc_after();
#pragma unroll
            for (int g = 0; g < NG; ++g) scores(g, 0);
            commit(BAR_KEMPTY);
        }
#pragma unroll 1
        for (int i = 0; i < n && ok; ++i) {
            const int s = i & 1, s1 = (i + 1) & 1;
            const bool more = i + 1 < n;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (g == 0) ok = wait(BAR_VFULL + s, i >> 1);
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    ok = ok && wait(BAR_PFULL + 2 * g + p, i);
                    if (!ok) break;
                    tc_after();
                    if (elect_one()) {
                        const u64 b = vd + (u32)(s * (P::VB >> 4) + p * (D * 128 / 16));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_ts(tmem + P::O0 + g * D, tmem + P::S0 + g * kTile + 32 * p + 8 * k, b + 2 * k, idesc_f16(D), p > 0 || k > 0 ? 1u : (u32)(i > 0));
                    }
                    __syncwarp();
                }
                if (ok && more) {
                    if (g == 0) ok = wait(BAR_KFULL + s1, (i + 1) >> 1);
                    if (ok) {
                        tc_after();
                        scores(g, s1);
                    }
                }
                if (!ok) break;
            }
            if (!ok) break;
            commit(BAR_VEMPTY + s);
            if (more) commit(BAR_KEMPTY + s1);
        }
        commit(BAR_O);
        // products in flight must end before TMEM is freed, also after an expired wait
        volatile int never = 0;
        mbar_wait_suspended(bar(BAR_O), 0, &never, &g_tcq_attention_error);
    }
    tc_before();
    __syncthreads();
    tc_after();
    // Back to the launch's registers for the code that all warps share: only behind the barrier, when every softmax warp has
    // had its larger share (a warp that took its registers back before could keep them from one forever).
    if (NG == 2) {
        if (warp < W_MMA) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 80;");
    }
    if (warp == W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::COLS) : "memory");
    if (splits == 1) return;

    // ---- the cluster's CTAs add their parts: each finishes a slice of the rows
    cluster_barrier();
    {
        constexpr int X = (D / 4) % 8 == 0 ? 7 : 3;
        const int rank = (int)cluster_rank(), rows = r1 - r0;
        const int s0 = rows * rank / splits, s1 = rows * (rank + 1) / splits;
        for (int e = tid; e < (s1 - s0) * (D / 8); e += P::THREADS) {
            const int row = s0 + e / (D / 8), c8 = e % (D / 8);
            float top = -INFINITY;
            for (int k = 0; k < splits; ++k) top = fmaxf(top, peer_ld2(peer_addr(sbase + P::ML0 + row * 8, k)).x);
            float acc[8] = {}, sum = 0.f;
            for (int k = 0; k < splits; ++k) {
                const float2 ml = peer_ld2(peer_addr(sbase + P::ML0 + row * 8, k));
                const float f = top == -INFINITY ? 0.f : ex2(ml.x - top);
                // Nothing of this part remains, unless its sum is NaN: scores that are NaN move no reference (a part of a NaN query
                // has -inf and a NaN sum), and the row has to say so.
                if (f == 0.f && ml.y == ml.y) continue;
                sum += ml.y * f;
                const u32 base = peer_addr(sbase, k) + row * (D * 4);
                const float4 u = peer_ld4(base + (((2 * c8) ^ (row & X)) << 4)), v = peer_ld4(base + (((2 * c8 + 1) ^ (row & X)) << 4));
                acc[0] += u.x * f, acc[1] += u.y * f, acc[2] += u.z * f, acc[3] += u.w * f;
                acc[4] += v.x * f, acc[5] += v.y * f, acc[6] += v.z * f, acc[7] += v.w * f;
            }
            const float f = sum != 0.f ? 1.f / sum : 0.f;
            u32 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = sum != 0.f ? pack2<DT>(acc[2 * j] * f, acc[2 * j + 1] * f) : 0u;
            const int r = r0 + row, tq = (int)fdiv((unsigned)r, A.by_group);
            u16* dst = A.out + (((i64)b * A.T + tq) * A.heads + h * A.group + r - tq * A.group) * D + 8 * c8;
            *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    cluster_barrier();
}

template <int DT, int D, int NG>
int launch_many(const AttnArgs& A, void* stream) {
    typedef Many<D, NG> P;
    const auto kern = k_attention_many<DT, D, NG>;
    const int R = A.T * A.group, row_tiles = (R + NG * kTile - 1) / (NG * kTile);
    const int tile_rows = ((R + row_tiles - 1) / row_tiles + 31) & ~31;            // even shares, in warps
    const i64 units = (i64)A.B * A.cache.kv_heads * row_tiles;
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
    // What a device can hold of clusters of 1 .. 8 CTAs, asked once per device.
    static std::atomic<int> held[64][9];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return TCQ_ERR_DEVICE;
    if (!held[dev][1].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P::BYTES) != cudaSuccess) return TCQ_ERR_LAUNCH;
        // the register shares of the roles are taken from what the launch gives the CTA: less would leave them waiting
        cudaFuncAttributes fa;
        if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess) return TCQ_ERR_LAUNCH;
        if (NG == 2 && fa.numRegs != P::LAUNCH_REGS) return TCQ_ERR_BUILD;
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
    // tiles, at least two tiles to a CTA of the longest sequence the table allows.
    int splits = 1;
    const i64 most = ((i64)A.blocks + 1) / 2;
    if (units < held[dev][1].load(std::memory_order_relaxed)) {
        double best = 1e30;
        for (int s = 1; s <= 8 && (s == 1 || 2 * s <= most); ++s) {
            const int n = held[dev][s].load(std::memory_order_relaxed);
            if (n <= 0) continue;
            const double cost = (double)((units + n - 1) / n) / s * (1 + 0.02 * (s - 1));
            if (cost < best) best = cost, splits = s;
        }
    }
    if (units * splits > 0x7fffffff) return TCQ_ERR_SHAPE;
    cfg.gridDim = dim3((unsigned)(units * splits));
    attr[0].val.clusterDim.x = splits;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, A, row_tiles, tile_rows, splits) == cudaSuccess ? TCQ_OK : TCQ_ERR_LAUNCH;
}

// Arrival counters at the head of the workspace, three per worker of the few-row kernel (its unit, and its two parts' groups).
// They are what has to be zero before the first call; TCQ_KV8_ZEROED_BYTES holds those of 455 SMs.
constexpr int kMostWarps = 12;
inline size_t counter_bytes(int sms) { return ((size_t)3 * kMostWarps * sms * sizeof(int) + 15) & ~(size_t)15; }

// ------------------------------------------------------------------------------------------------ host side
}  // namespace

extern "C" {

// Rows that the few-row kernel takes: two tiles of 8, or four where they fit the registers (head widths up to 64).
static inline bool few_rows(i64 rows, int head_dim) { return rows <= 16 || (rows <= 32 && head_dim <= 64); }

size_t tcq_kv8_attention_workspace(int B, int T, int heads, int kv_heads, int head_dim, int blocks) {
    if (B < 1 || T < 1 || heads < 1 || kv_heads < 1 || head_dim < 1 || blocks < 1 || heads % kv_heads) return 0;
    const int sms = tcq_sm_count();
    const i64 rows = (i64)T * (heads / kv_heads);
    if (few_rows(rows, head_dim)) return counter_bytes(sms) + (size_t)2 * kMostWarps * sms * ((rows + 7) / 8 * 8) * (head_dim + 2) * sizeof(float);
    return 16;
}

int tcq_kv8_attention(const tcq_kv8_cache* cache, const void* q, int dtype, int64_t q_sb, int64_t q_st, void* out, const int32_t* table,
                      int blocks, const int32_t* lens, const int32_t* count, int causal, float scale, int B, int T, int heads,
                      void* workspace, size_t workspace_bytes, void* stream) {
    const int e = check_cache(cache);
    if (e) return e;
    if (!q || !out || !table || !lens) return TCQ_ERR_ARG;
    if (dtype != TCQ_DT_BF16 && dtype != TCQ_DT_F16) return TCQ_ERR_DTYPE;
    const int Hk = cache->kv_heads;
    if (B < 1 || T < 1 || blocks < 1 || heads < 1 || heads % Hk || blocks > (0x7fffffff / kBlk)) return TCQ_ERR_SHAPE;
    if ((i64)B * Hk > 0x7fffffff || (i64)B * Hk * (blocks + 1) > 0x7fffffff) return TCQ_ERR_SHAPE;
    if (!tcq_aligned(q, 16) || !tcq_aligned(out, 16) || ((q_sb | q_st) & 7)) return TCQ_ERR_ALIGN;
    if (counter_bytes(tcq_sm_count()) > TCQ_KV8_ZEROED_BYTES) return TCQ_ERR_DEVICE;
    if (!workspace || workspace_bytes < tcq_kv8_attention_workspace(B, T, heads, Hk, cache->head_dim, blocks)) return TCQ_ERR_WORKSPACE;
    const int sms = tcq_sm_count();
    AttnArgs A = {*cache, (const u16*)q, q_sb, q_st, (u16*)out, table, lens, count, nullptr, (int*)workspace, blocks, causal, B, T, heads,
                  heads / Hk, make_fastdiv((unsigned)(heads / Hk)), scale * 1.4426950408889634f};
    const i64 rows = (i64)T * A.group;
    if (few_rows(rows, cache->head_dim)) {
        A.part = reinterpret_cast<float*>((char*)workspace + counter_bytes(sms));
        const i64 units = (i64)B * Hk;
        // Many short sequences: whole units to a warp, nothing to add up (1024 units of three pages: see the kernel).
        const int whole = blocks <= 8 && units >= 2 * sms;
        return by_head_dim(cache->head_dim, [&](auto d) {
            constexpr int D = decltype(d)::value;
            auto go = [&](auto tiles) {
                constexpr int NT = decltype(tiles)::value;
                typedef Few<D, NT> P;
                return dtype == TCQ_DT_BF16 ? launch_big<k_attention_few<TCQ_DT_BF16, D, NT>>(dim3(sms), P::WARPS * 32, P::BYTES, stream, A, whole)
                                            : launch_big<k_attention_few<TCQ_DT_F16, D, NT>>(dim3(sms), P::WARPS * 32, P::BYTES, stream, A, whole);
            };
            if constexpr (D <= 64) {
                if (rows > 24) return go(std::integral_constant<int, 4>());
                if (rows > 16) return go(std::integral_constant<int, 3>());
            }
            return rows > 8 ? go(std::integral_constant<int, 2>()) : go(std::integral_constant<int, 1>());
        });
    }
    if (rows > 0x7fffffff) return TCQ_ERR_SHAPE;
    return by_head_dim(cache->head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (dtype == TCQ_DT_BF16) return rows <= kTile ? launch_many<TCQ_DT_BF16, D, 1>(A, stream) : launch_many<TCQ_DT_BF16, D, 2>(A, stream);
        return rows <= kTile ? launch_many<TCQ_DT_F16, D, 1>(A, stream) : launch_many<TCQ_DT_F16, D, 2>(A, stream);
    });
}

}  // extern "C"
