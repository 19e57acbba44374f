// Attention over the 8-bit cache.
#include <type_traits>

#include "memory.cuh"

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
TCQ_HD int page_of(const int* row, int blk, int pages) {
    const int p = row[blk];
    if ((unsigned)p >= (unsigned)pages) {
        out_of_range();
        return p < 0 ? 0 : pages - 1;
    }
    return p;
}

// ------------------------------------------------------------------------------------------------ few query rows
// T * group <= 16 MT query rows share a key head (single tokens, short action sequences): the kernel streams the pages once and
// is bound by HBM.
//
// Mathematics. With integers k, v and block scales ks, vs: score x = (q . k) ks scale log2(e) + log2(vs), reference m >= x - 4,
// weight p = 2^(x - m + 10); out = sum p v / sum (p / vs). Folding vs into the exponent keeps every product operand an exact
// small integer or one rounding of p, and the sum of p is formed before that rounding. m moves only when a score passes it
// by more than 2^4, so the accumulators are rarely rescaled. Operands are FP16: an int8 is exact, a query row is scaled by a
// power of two so that its largest element lies in [2^14, 2^15) (elements below 2^-28 of it lose bits, those of BF16
// inputs above that lose none), and p <= 2^14 keeps 11 bits down to 2^-28 of the largest and is dropped below 2^-38.
//
// Layout. A warp takes whole pages. S = Q K^T and O = P V are m16n8k16 products. The order of a contraction is free, so lane
// (n, t) reads 16 consecutive bytes of key row n (or of value row n: 16 tokens) and feeds them to four products: one 16-byte
// shared load per 16 elements and no transposition. Key columns are assigned to score columns so that a lane's scores are
// exactly the tokens whose values it reads: key(block 2 i + h, column 2 t + e) = 16 t + 4 i + 2 h + e.
//
// int8 -> FP16: u = byte ^ 0x80, 0x6400 | u is 1024 + u, minus 1152: five instructions for four elements.

constexpr int kWarps = 8;
constexpr float kRef = 10.f;          // log2 of the weight of a score equal to the reference
constexpr float kSlack = 4.f;         // growth of the maximum that does not move the reference

TCQ_HD float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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
    int blocks, causal, B, T, heads, group, workers;
    float scale_log2;      // scale * log2(e)
};

// Shared-memory plan of the few-row kernel: a ring of NH half pages (64 D bytes: a block's keys or its values) per warp.
template <int D, int MT, int W>
struct Few {
    static constexpr int HALF = kBlk * D;
    static constexpr int NH = D <= 48 ? 8 : D == 64 ? 6 : D == 80 ? 5 : D == 96 ? 4 : 3;
    static constexpr int PAD = D == 128 ? 4 : 8;
    static constexpr int RING = kWarps * NH * HALF;
    static constexpr int HDR = RING;                                       // ks, vs of each half page
    static constexpr int ML = HDR + kWarps * NH * 8;                       // m, l of every warp and row
    static constexpr int MERGE = ML + (W > 1 ? kWarps * 16 * MT * 8 : 0);  // one group of 8 rows of every warp
    static constexpr int BYTES = MERGE + (W > 1 ? kWarps * 8 * (D + PAD) * 4 : 0);
};

// 16-byte chunk c of key row r lies at chunk c ^ swap(r): rows of 128 bytes put their halves on alternating banks.
template <int D>
TCQ_HD int key_chunk(int r, int c) { return D == 128 ? c ^ ((r & 1) << 2) : c; }

// A position in the flattened list of pages: sequence b, key head h, unit (b, h) begins at ubeg and takes vp places, of which
// the first np are pages.
struct Place {
    int b, h, ubeg, vp, np;
};

template <int DT, int D, int MT, int W>
__global__ void __launch_bounds__(kWarps * 32, 1) k_attention_few(const AttnArgs A) {
    typedef Few<D, MT, W> P;
    constexpr int NH = P::NH, KS = D / 16, ROWS = 16 * MT;
    extern __shared__ __align__(16) char smem[];
    __shared__ int s_scan[kWarps + 4];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = lane >> 2, t = lane & 3;
    const int Hk = A.cache.kv_heads, R = A.T * A.group;
    char* ring = smem + warp * NH * P::HALF;
    float2* hdr = reinterpret_cast<float2*>(smem + P::HDR) + warp * NH;

    // ---- this worker's range [x0, x1) of places, and where it begins
    int align = 1, chunk = 1, x0, x1;
    Place at;
    auto places = [&](int len) { return max(1, (len + kBlk - 1) / kBlk); };
    auto round_up = [&](int v) { return (v + align - 1) / align * align; };
    if (W == 1) {
        // whole units, one after the other
        const int u = blockIdx.x * kWarps + warp;
        if (u >= A.B * Hk) return;
        at.b = u / Hk, at.h = u - at.b * Hk;
        x0 = 0, x1 = 1 << 30;
    } else {
        // all sequences' lengths: every thread a run of them, summed over the block
        const int per = (A.B + kWarps * 32 - 1) / (kWarps * 32), b0 = min(A.B, tid * per), b1 = min(A.B, b0 + per);
        int pages = 0, seqs = 0;
        for (int b = b0; b < b1; ++b) pages += places(tokens_of(A.lens, b, A.blocks)), ++seqs;
        int total = pages;
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (lane == 0) s_scan[warp] = total;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) total += s_scan[w];
        __syncthreads();
        // few pages: places in groups of one page per warp, so that a worker serves one unit
        if ((i64)total * Hk <= (i64)kWarps * A.workers) align = kWarps;
        int mine = 0;
        for (int b = b0; b < b1; ++b) mine += round_up(places(tokens_of(A.lens, b, A.blocks)));
        int scan = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) s_scan[warp] = scan;
        __syncthreads();
        int before = scan - mine, all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            before += w < warp ? s_scan[w] : 0;
            all += s_scan[w];
        }
        all *= Hk;
        chunk = round_up((all + A.workers - 1) / A.workers);
        x0 = min((i64)blockIdx.x * chunk, (i64)all), x1 = min(x0 + chunk, all);
        if (x0 >= x1) return;                                             // the whole block
        int off = before * Hk;
        for (int b = b0; b < b1; ++b) {
            const int w = round_up(places(tokens_of(A.lens, b, A.blocks))) * Hk;
            if (x0 >= off && x0 < off + w) s_scan[kWarps] = b, s_scan[kWarps + 1] = off;
            off += w;
        }
        __syncthreads();
        at.b = s_scan[kWarps];
        const int vp = round_up(places(tokens_of(A.lens, at.b, A.blocks)));
        at.h = (x0 - s_scan[kWarps + 1]) / vp;
        at.ubeg = s_scan[kWarps + 1] + at.h * vp;
    }
    auto measure = [&](Place& p) {
        const int len = tokens_of(A.lens, p.b, A.blocks);
        p.np = (len + kBlk - 1) / kBlk;
        p.vp = round_up(max(1, p.np));
    };
    measure(at);
    if (W == 1) at.ubeg = 0, x1 = at.vp;
    // The next unit of the range; false at its end.
    auto next_unit = [&](Place& p, int& end) -> bool {
        if (W == 1) {
            const int u = p.b * Hk + p.h + A.workers * kWarps;
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
    int px = x0 + (W == 1 ? 0 : warp), pend = x1, pid = 0, pslot = 0;
    bool pmore = true;
    auto p_settle = [&]() {                      // move px to the warp's next place that is a page
        for (;;) {
            if (px >= min(pat.ubeg + pat.vp, pend)) {
                if (!next_unit(pat, pend)) {
                    pmore = false;
                    return;
                }
                if (W == 1) px = 0;
                continue;
            }
            if (px - pat.ubeg < pat.np) break;
            px += W;
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
                px += W;
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
    int x = x0 + (W == 1 ? 0 : warp);
    for (;;) {
        const int len = tokens_of(A.lens, at.b, A.blocks), cnt = queries_of(A.count, at.b, A.T);
        // query rows r = t * group + g of this head, as FP16 fragments scaled by a power of two
        u32 qa[MT][KS][4];
        float crow[MT][2];
        int limit[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int r = 16 * mt + 8 * hf + n, tq = r / A.group, g = r - tq * A.group;
                const bool live = r < R && tq < cnt;
                limit[mt][hf] = !live ? 0 : A.causal ? min(max(len - cnt + tq + 1, 0), len) : len;
                const u16* qr = A.q + at.b * A.q_sb + tq * A.q_st + (i64)(at.h * A.group + g) * D;
                float v[KS][4], amax = 0.f;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    // the four elements that lane t contributes to step s (see the key loads)
                    const int d = s < D / 64 * 4 ? 64 * (s / 4) + 16 * t + 4 * (s % 4)
                                : s < D / 32 * 2 ? D / 64 * 64 + 8 * t + 4 * (s - D / 64 * 4) : D / 32 * 32 + 4 * t;
                    uint2 w = live ? *reinterpret_cast<const uint2*>(qr + d) : make_uint2(0u, 0u);
                    unpack2<DT>(w.x, v[s][0], v[s][1]);
                    unpack2<DT>(w.y, v[s][2], v[s][3]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(v[s][e]));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                float back;
                const float up = row_scale(amax, back);
                crow[mt][hf] = back * A.scale_log2;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    qa[mt][s][hf] = half2_of(v[s][0] * up, v[s][1] * up);
                    qa[mt][s][2 + hf] = half2_of(v[s][2] * up, v[s][3] * up);
                }
            }
        const int open = A.causal ? len - cnt + 1 : len;         // keys below this are seen by every query
        float o[MT][D / 8][4], m[MT][2], l[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.f;
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.f;
        }
        const int seg_end = min(at.ubeg + at.vp, end);
#pragma unroll 1
        for (; x < seg_end; x += W) {
            const int pg = x - at.ubeg;
            if (pg >= at.np) continue;
            const float2* sp = hdr + slot;
            const char* kp = take();
            const float2 sc = *sp;
            slot = slot + 1 == NH ? 0 : slot + 1;
            float s[MT][8][4];
#pragma unroll
            for (int nb = 0; nb < 8; ++nb) {
                const int r = 16 * (n >> 1) + 2 * nb + (n & 1);           // nb = 2 i + h: 4 i + 2 h = 2 nb
                const char* row = kp + r * D;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][nb][0] = s[mt][nb][1] = s[mt][nb][2] = s[mt][nb][3] = 0.f;
                auto step = [&](int ks, u32 w) {
                    u32 b0, b1;
                    int8x4_to_half(w, b0, b1);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) mma16816(s[mt][nb], qa[mt][ks][0], qa[mt][ks][1], qa[mt][ks][2], qa[mt][ks][3], b0, b1);
                };
#pragma unroll
                for (int q4 = 0; q4 < D / 64; ++q4) {
                    const uint4 w = *reinterpret_cast<const uint4*>(row + key_chunk<D>(r, 4 * q4 + t) * 16);
                    step(4 * q4, w.x), step(4 * q4 + 1, w.y), step(4 * q4 + 2, w.z), step(4 * q4 + 3, w.w);
                }
                if (D % 64 >= 32) {
                    const uint2 w = *reinterpret_cast<const uint2*>(row + D / 64 * 64 + 8 * t);
                    step(D / 64 * 4, w.x), step(D / 64 * 4 + 1, w.y);
                }
                if (D % 32) step(D / 32 * 2, *reinterpret_cast<const u32*>(row + D / 32 * 32 + 4 * t));
            }
            const float vs = safe_scale(sc.y), bias = lg2(vs), inv = 1.f / vs;
            const bool masked = (pg + 1) * kBlk > open;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    if (16 * mt + 8 * hf >= R) continue;
                    const float c = crow[mt][hf] * sc.x;
                    float top = -INFINITY;
                    if (masked) {
                        const int lim = limit[mt][hf] - pg * kBlk - 16 * t;
#pragma unroll
                        for (int nb = 0; nb < 8; ++nb)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float& v = s[mt][nb][2 * hf + e];
                                v = 2 * nb + e < lim ? __fmaf_rn(v, c, bias) : -INFINITY;
                                top = fmaxf(top, v);
                            }
                    } else {
#pragma unroll
                        for (int nb = 0; nb < 8; ++nb)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float& v = s[mt][nb][2 * hf + e];
                                v = __fmaf_rn(v, c, bias);
                                top = fmaxf(top, v);
                            }
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    float& mr = m[mt][hf];
                    const bool move = top > mr + kSlack;
                    if (__any_sync(0xffffffffu, move)) {
                        const float f = move ? ex2(mr - top) : 1.f;
                        if (move) mr = top;
                        l[mt][hf] *= f;
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) o[mt][i][2 * hf] *= f, o[mt][i][2 * hf + 1] *= f;
                    }
                    const float base = (mr == -INFINITY ? 0.f : mr) - kRef;
                    float sum = 0.f;
#pragma unroll
                    for (int nb = 0; nb < 8; ++nb)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float& v = s[mt][nb][2 * hf + e];
                            v = ex2(v - base);
                            sum += v;
                        }
                    l[mt][hf] = __fmaf_rn(sum, inv, l[mt][hf]);
                }
            if (sc.y < kLeastScale) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nb = 0; nb < 8; ++nb) s[mt][nb][0] = s[mt][nb][1] = s[mt][nb][2] = s[mt][nb][3] = 0.f;
            }
            u32 pa[MT][4][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool high = 16 * mt + 8 < R;
                    pa[mt][i][0] = half2_of(s[mt][2 * i][0], s[mt][2 * i][1]);
                    pa[mt][i][1] = high ? half2_of(s[mt][2 * i][2], s[mt][2 * i][3]) : 0u;
                    pa[mt][i][2] = half2_of(s[mt][2 * i + 1][0], s[mt][2 * i + 1][1]);
                    pa[mt][i][3] = high ? half2_of(s[mt][2 * i + 1][2], s[mt][2 * i + 1][3]) : 0u;
                }
            const char* vp = take();
            slot = slot + 1 == NH ? 0 : slot + 1;
#pragma unroll
            for (int db = 0; db < D / 8; ++db) {
                const uint4 w = *reinterpret_cast<const uint4*>(vp + (8 * db + n) * kBlk + 16 * t);
                const u32 ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u32 b0, b1;
                    int8x4_to_half(ww[i], b0, b1);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) mma16816(o[mt][db], pa[mt][i][0], pa[mt][i][1], pa[mt][i][2], pa[mt][i][3], b0, b1);
                }
            }
        }
        // ---- the unit's rows, or this worker's part of them
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                float& v = l[mt][hf];
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                if (limit[mt][hf] == 0) v = 0.f;              // a row that sees no token
            }
        auto out_row = [&](int r) -> u16* {
            const int tq = r / A.group;
            return A.out + (((i64)at.b * A.T + tq) * A.heads + at.h * A.group + r - tq * A.group) * D;
        };
        if (W == 1) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int r = 16 * mt + 8 * hf + n;
                    if (r >= R) continue;
                    const float f = l[mt][hf] != 0.f ? 1.f / l[mt][hf] : 0.f;
                    u32* dst = reinterpret_cast<u32*>(out_row(r));
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) dst[4 * i + t] = pack2<DT>(o[mt][i][2 * hf] * f, o[mt][i][2 * hf + 1] * f);
                }
        } else {
            float2* ml = reinterpret_cast<float2*>(smem + P::ML);
            float* buf = reinterpret_cast<float*>(smem + P::MERGE);
            constexpr int ST = D + P::PAD;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    if (t == 0) ml[warp * ROWS + 16 * mt + 8 * hf + n] = make_float2(m[mt][hf], l[mt][hf]);
            __syncthreads();
            const bool whole = max(at.ubeg, x0) == at.ubeg && seg_end == at.ubeg + at.vp;
            const int first = at.ubeg / chunk, last = (at.ubeg + at.vp - 1) / chunk, me = blockIdx.x;
            float* part = A.part + (i64)(2 * me + (me == first ? 1 : 0)) * ROWS * (D + 2);
#pragma unroll
            for (int grp = 0; grp < 2 * MT; ++grp) {
                if (8 * grp >= R) break;
                const int mt = grp >> 1, hf = grp & 1;
                {
                    float top = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * ROWS + 8 * grp + n].x);
                    const float f = top == -INFINITY ? 0.f : ex2(m[mt][hf] - top);
#pragma unroll
                    for (int i = 0; i < D / 8; ++i)
                        *reinterpret_cast<float2*>(buf + (warp * 8 + n) * ST + 8 * i + 2 * t) =
                            make_float2(o[mt][i][2 * hf] * f, o[mt][i][2 * hf + 1] * f);
                }
                __syncthreads();
                const int rows = min(8, R - 8 * grp);
                for (int i = tid; i < rows * (D / 2); i += kWarps * 32) {
                    const int rr = i / (D / 2), d = (i - rr * (D / 2)) * 2, r = 8 * grp + rr;
                    float top = -INFINITY, sum = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * ROWS + r].x);
                    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float2 v = *reinterpret_cast<const float2*>(buf + (w * 8 + rr) * ST + d), e = ml[w * ROWS + r];
                        acc.x += v.x, acc.y += v.y;
                        sum += e.y * (top == -INFINITY ? 0.f : ex2(e.x - top));
                    }
                    if (whole) {
                        const float f = sum != 0.f ? 1.f / sum : 0.f;
                        *reinterpret_cast<u32*>(out_row(r) + d) = pack2<DT>(acc.x * f, acc.y * f);
                    } else {
                        *reinterpret_cast<float2*>(part + r * (D + 2) + d) = acc;
                        if (d == 0) *reinterpret_cast<float2*>(part + r * (D + 2) + D) = make_float2(top, sum);
                    }
                }
                __syncthreads();
            }
            if (!whole) {
                // the last of the unit's workers adds the parts in their order
                __threadfence();
                __syncthreads();
                if (tid == 0) {
                    const int seen = atomicAdd(A.counters + first, 1);
                    s_scan[kWarps + 3] = seen == last - first;
                    if (seen == last - first) A.counters[first] = 0;
                }
                __syncthreads();
                if (s_scan[kWarps + 3]) {
                    __threadfence();
                    for (int i = tid; i < R * (D / 2); i += kWarps * 32) {
                        const int r = i / (D / 2), d = (i - r * (D / 2)) * 2;
                        float top = -INFINITY;
                        for (int w = first; w <= last; ++w) {
                            const float* p = A.part + (i64)(2 * w + (w == first ? 1 : 0)) * ROWS * (D + 2) + r * (D + 2);
                            top = fmaxf(top, __ldcg(p + D));
                        }
                        float sum = 0.f;
                        float2 acc = make_float2(0.f, 0.f);
                        for (int w = first; w <= last; ++w) {
                            const float* p = A.part + (i64)(2 * w + (w == first ? 1 : 0)) * ROWS * (D + 2) + r * (D + 2);
                            const float2 e = __ldcg(reinterpret_cast<const float2*>(p + D)), v = __ldcg(reinterpret_cast<const float2*>(p + d));
                            const float f = top == -INFINITY ? 0.f : ex2(e.x - top);
                            acc.x += v.x * f, acc.y += v.y * f;
                            sum += e.y * f;
                        }
                        const float f = sum != 0.f ? 1.f / sum : 0.f;
                        *reinterpret_cast<u32*>(out_row(r) + d) = pack2<DT>(acc.x * f, acc.y * f);
                    }
                }
                __syncthreads();
            }
        }
        if (!next_unit(at, end)) break;
        if (W == 1) x = 0;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// One warp per query row (sequence, query, head), 32 keys at a time: each lane forms one score (its key's row of D bytes),
// the warp updates the running maximum and sum, and each lane then adds the keys' values into its own elements d = lane + 32 i.
template <int DT, int D>
__global__ void __launch_bounds__(128) k_attention_rows(tcq_kv8_cache cache, const u16* __restrict__ q, i64 q_sb, i64 q_st, u16* __restrict__ out,
                                                        const int* __restrict__ table, int blocks, const int* __restrict__ lens,
                                                        const int* __restrict__ count, int causal, float scale, i64 rows, int T, int heads) {
    __shared__ float sq[4][D], sp[4][32];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const i64 row = (i64)blockIdx.x * 4 + warp;
    if (row >= rows) return;
    const int h = (int)(row % heads);
    const i64 bt = row / heads, b = bt / T;
    const int t = (int)(bt - b * T), Hk = cache.kv_heads, hk = h / (heads / Hk);
    const int len = tokens_of(lens, b, blocks), cnt = queries_of(count, b, T);
    const int limit = t >= cnt ? 0 : causal ? min(max(len - cnt + t + 1, 0), len) : len;
    for (int d = lane; d < D; d += 32) sq[warp][d] = elem_f<DT>(q[b * q_sb + t * q_st + (i64)h * D + d]) * scale;
    __syncwarp();
    constexpr int ND = (D + 31) / 32;
    float o[ND] = {}, m = -INFINITY, l = 0.f;
    for (int k0 = 0; k0 < limit; k0 += 32) {
        const i64 ph = (i64)page_of(table + b * blocks, k0 / kBlk, cache.pages) * Hk + hk, off = ph * (kBlk * D);
        const int slot = k0 % kBlk;
        const i8* kr = cache.k + off + (slot + lane) * D;
        float s = 0.f;
        for (int d = 0; d < D; d += 4) {
            const u32 w = *reinterpret_cast<const u32*>(kr + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fmaf((float)(int)(i8)(w >> (8 * e)), sq[warp][d + e], s);
        }
        s *= cache.k_scale[ph];
        if (k0 + lane >= limit) s = -INFINITY;
        float top = s;
#pragma unroll
        for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float mn = fmaxf(m, top), f = expf(m - mn), p = expf(s - mn);
        m = mn;
        sp[warp][lane] = p * cache.v_scale[ph];
        float sum = p;
#pragma unroll
        for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        l = fmaf(l, f, sum);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            const int d = lane + 32 * i;
            if (d >= D) break;
            const u32* vr = reinterpret_cast<const u32*>(cache.v + off + d * kBlk + slot);
            float a = o[i] * f;
            for (int j = 0; j < 8; ++j) {
                const u32 w = vr[j];
#pragma unroll
                for (int e = 0; e < 4; ++e) a = fmaf(sp[warp][4 * j + e], (float)(int)(i8)(w >> (8 * e)), a);
            }
            o[i] = a;
        }
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        const int d = lane + 32 * i;
        if (d < D) out[(bt * heads + h) * D + d] = (u16)pack2<DT>(l > 0.f ? o[i] / l : 0.f, 0.f);
    }
}

// Arrival counters at the head of the workspace, one per worker.
inline size_t counter_bytes(int workers) { return ((size_t)workers * sizeof(int) + 15) & ~(size_t)15; }

// ------------------------------------------------------------------------------------------------ host side
}  // namespace

extern "C" {

// Rows that the few-row kernel takes: one m16 tile, or two where both fit the registers (head widths up to 64).
static inline bool few_rows(i64 rows, int head_dim) { return rows <= 16 || (rows <= 32 && head_dim <= 64); }

size_t tcq_kv8_attention_workspace(int B, int T, int heads, int kv_heads, int head_dim, int blocks) {
    if (B < 1 || T < 1 || heads < 1 || kv_heads < 1 || head_dim < 1 || blocks < 1 || heads % kv_heads) return 0;
    const int sms = tcq_sm_count();
    const i64 rows = (i64)T * (heads / kv_heads);
    if (few_rows(rows, head_dim)) return counter_bytes(sms) + (size_t)2 * sms * (rows <= 16 ? 16 : 32) * (head_dim + 2) * sizeof(float);
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
    if ((i64)B * Hk > 0x7fffffff || (i64)B * Hk * (blocks + kWarps) > 0x7fffffff) return TCQ_ERR_SHAPE;
    if (!tcq_aligned(q, 16) || !tcq_aligned(out, 16) || ((q_sb | q_st) & 7)) return TCQ_ERR_ALIGN;
    if (!workspace || workspace_bytes < tcq_kv8_attention_workspace(B, T, heads, Hk, cache->head_dim, blocks)) return TCQ_ERR_WORKSPACE;
    const int sms = tcq_sm_count();
    AttnArgs A = {*cache, (const u16*)q, q_sb, q_st, (u16*)out, table, lens, count, nullptr, (int*)workspace, blocks, causal, B, T, heads,
                  heads / Hk, sms, scale * 1.4426950408889634f};
    const i64 rows = (i64)T * A.group;
    if (few_rows(rows, cache->head_dim)) {
        A.part = reinterpret_cast<float*>((char*)workspace + counter_bytes(sms));
        const i64 units = (i64)B * Hk;
        // Short sequences of many units: a warp per unit, nothing to merge.
        const bool alone = blocks <= 8 && units >= 2 * sms;
        const int grid = alone ? (int)((units + kWarps - 1) / kWarps < sms ? (units + kWarps - 1) / kWarps : sms) : sms;
        if (alone) A.workers = grid;
        return by_head_dim(cache->head_dim, [&](auto d) {
            constexpr int D = decltype(d)::value;
            auto go = [&](auto bf, auto one) {
                constexpr int DT = decltype(bf)::value ? TCQ_DT_BF16 : TCQ_DT_F16, W = decltype(one)::value ? 1 : kWarps;
                if constexpr (D <= 64) {
                    if (rows > 16) return launch_big<k_attention_few<DT, D, 2, W>>(dim3(grid), kWarps * 32, Few<D, 2, W>::BYTES, stream, A);
                }
                return launch_big<k_attention_few<DT, D, 1, W>>(dim3(grid), kWarps * 32, Few<D, 1, W>::BYTES, stream, A);
            };
            const std::true_type yes{};
            const std::false_type no{};
            return dtype == TCQ_DT_BF16 ? (alone ? go(yes, yes) : go(yes, no)) : (alone ? go(no, yes) : go(no, no));
        });
    }
    const i64 all = (i64)B * T * heads;
    if ((all + 3) / 4 > 0x7fffffff) return TCQ_ERR_SHAPE;
    return by_head_dim(cache->head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_pdl(dtype == TCQ_DT_BF16 ? k_attention_rows<TCQ_DT_BF16, D> : k_attention_rows<TCQ_DT_F16, D>,
                          dim3((unsigned)((all + 3) / 4)), 128, 0, stream, *cache, (const u16*)q, (i64)q_sb, (i64)q_st, (u16*)out, table,
                          blocks, lens, count, causal, scale, all, T, heads);
    });
}

}  // extern "C"
