// Streaming-memory kernels around the attention: the rotary embedding with several axes, writing new tokens into the 8-bit
// cache, and reading the cache back as values.
#include <type_traits>

#include "memory.cuh"

__device__ int g_tcq_memory_error;

int tcq_memory_error(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tcq_memory_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && v) {
        const int z = 0;
        if (cudaMemcpyToSymbol(g_tcq_memory_error, &z, sizeof(int)) != cudaSuccess) return -1;
    }
    return v;
}

namespace {

using namespace tcq;

// ------------------------------------------------------------------------------------------------ rotary, several axes
// A unit is V frequencies of one head: 2 V elements, as two V-element vectors (half-split: j and j + D/2; pairs: 2 V
// neighbours). A thread keeps its V cosines and sines of one token in registers and turns that unit of every hp-th head,
// so the tables are read once per token and 2 V / (heads / hp) elements. Bound by HBM (many tokens) or latency (few).
template <int BYTES> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef u32 type; };
template <> struct Raw<2> { typedef u16 type; };

template <int DT, int V>
struct Vec {
    static constexpr int BYTES = V * (DT == TCQ_DT_F32 ? 4 : 2);
    typedef typename Raw<BYTES>::type R;
    static TCQ_HD void load(const void* p, float* v) { unpack(*reinterpret_cast<const R*>(p), v); }
    static TCQ_HD void unpack(R r, float* v) {
        union { R r; u32 w[(BYTES + 3) / 4]; u16 h[BYTES / 2]; } u;
        u.r = r;
        if (DT == TCQ_DT_F32) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = __uint_as_float(u.w[i]);
        } else if (V == 1) {
            v[0] = elem_f<DT>(u.h[0]);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) unpack2<DT>(u.w[i], v[2 * i], v[2 * i + 1]);
        }
    }
    static TCQ_HD void store(void* p, const float* v) {
        union { R r; u32 w[(BYTES + 3) / 4]; u16 h[BYTES / 2]; } u;
        if (DT == TCQ_DT_F32) {
#pragma unroll
            for (int i = 0; i < V; ++i) u.w[i] = __float_as_uint(v[i]);
        } else if (V == 1) {
            u.h[0] = (u16)pack2<DT>(v[0], 0.f);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) u.w[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
        }
        *reinterpret_cast<R*>(p) = u.r;
    }
};

template <int DT, int V, bool PAIRS, int HB>
__global__ void __launch_bounds__(256, 3) k_rope_axes(const char* __restrict__ x, char* __restrict__ out, RopeArgs r, i64 x_sb, i64 x_st,
                                                   i64 o_sb, i64 o_st, i64 rows, int T, int heads, int C, int hp, float sign) {
    constexpr int E = DT == TCQ_DT_F32 ? 4 : 2;
    pdl_launch_dependents();
    pdl_wait();
    const int per = C * hp;
    const i64 row = (i64)blockIdx.x * (blockDim.x / per) + threadIdx.x / per;
    if (row >= rows) return;
    const int u = threadIdx.x % per, c = u % C, h0 = u / C;
    const i64 b = row / T, t = row - b * T;
    const int D = 2 * r.half, first = PAIRS ? 2 * V * c : V * c, second = PAIRS ? first + V : first + r.half;
    const char* xr = x + (b * x_sb + t * x_st) * E;
    char* orow = out + (b * o_sb + t * o_st) * E;
    // HB > 1: that many heads are requested before the tables, whose loads wait for the positions
    typedef typename Vec<DT, V>::R Rv;
    float cs[V], sn[V];
    auto tables = [&]() {
        rope_cs<V>(r, row, V * c, cs, sn, &g_tcq_memory_error);
#pragma unroll
        for (int i = 0; i < V; ++i) sn[i] *= sign;
    };
    if (HB == 1) tables();
#pragma unroll 1
    for (int hb = h0; hb < heads; hb += HB * hp) {
        Rv lo[HB], hi[HB];
#pragma unroll
        for (int k = 0; k < HB; ++k)
            if (hb + k * hp < heads) {
                lo[k] = *reinterpret_cast<const Rv*>(xr + (i64)((hb + k * hp) * D + first) * E);
                hi[k] = *reinterpret_cast<const Rv*>(xr + (i64)((hb + k * hp) * D + second) * E);
            }
        if (HB > 1 && hb == h0) tables();
#pragma unroll
        for (int k = 0; k < HB; ++k)
            if (hb + k * hp < heads) {
                float a[2 * V];
                Vec<DT, V>::unpack(lo[k], a);
                Vec<DT, V>::unpack(hi[k], a + V);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (PAIRS) turn(a[2 * i], a[2 * i + 1], cs[i], sn[i]);
                    else turn(a[i], a[V + i], cs[i], sn[i]);
                }
                Vec<DT, V>::store(orow + (i64)((hb + k * hp) * D + first) * E, a);
                Vec<DT, V>::store(orow + (i64)((hb + k * hp) * D + second) * E, a + V);
            }
    }
}

template <int DT, int V>
int launch_rope(const void* x, void* out, const RopeArgs& r, i64 x_sb, i64 x_st, i64 o_sb, i64 o_st, int B, int T, int heads, bool pairs,
                float sign, void* stream) {
    const int C = r.half / V;                      // units of a head (at most 128)
    const i64 rows = (i64)B * T;
    // Heads side by side: all of them while the launch is short of threads (latency), a quarter of them when it has many
    // (four heads share a thread's cosines and sines: 2 x 8191 x 32 x 128 F16 71 -> 59 us).
    int hp = heads < 256 / C ? heads : 256 / C;
    const bool four = heads >= 4 && rows * C * heads > (i64)tcq_sm_count() * 2048;
    if (four && (heads + 4 - 1) / 4 < hp) hp = (heads + 4 - 1) / 4;
    const int tokens = 256 / (C * hp);             // tokens of a block
    const i64 blocks = (rows + tokens - 1) / tokens;
    if (blocks > 0x7fffffff) return TCQ_ERR_SHAPE;
    const auto kern = pairs ? (four ? k_rope_axes<DT, V, true, 4> : k_rope_axes<DT, V, true, 1>)
                            : (four ? k_rope_axes<DT, V, false, 4> : k_rope_axes<DT, V, false, 1>);
    return launch_pdl(kern, dim3((unsigned)blocks), tokens * C * hp, 0, stream,
                      (const char*)x, (char*)out, r, x_sb, x_st, o_sb, o_st, rows, T, heads, C, hp, sign);
}

// ------------------------------------------------------------------------------------------------ cache append
// Four quotients x * inv, |x * inv| < 127.5, rounded to nearest even and packed: 1.5 * 2^23 added leaves the integer in a
// float's low bits.
TCQ_HD u32 q8x4(const float* x, float inv) {
    u32 b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(x[i] * inv + 12582912.f);
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}
// The rare block with infinities or NaN: infinities become the block's largest value, NaN zero.
TCQ_HD float tamed(float x, float s) { return x == x ? fminf(fmaxf(x, -127.f * s), 127.f * s) : 0.f; }

// Largest magnitudes of 16-bit elements, two at a time: without their signs they order as unsigned integers, NaN above all.
TCQ_HD u32 max2(u32 m, u32 w) { return __vmaxu2(m, w & 0x7fff7fffu); }
TCQ_HD u32 max2(u32 m, const uint4& w) { return max2(max2(max2(max2(m, w.x), w.y), w.z), w.w); }
template <int DT>
TCQ_HD u32 max2_bits(u32 m) { return __float_as_uint(elem_f<DT>((u16)max(m & 0xffffu, m >> 16))); }

TCQ_HD u32 requant4(u32 w, float ratio) {
    u32 o = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) o |= (u32)(__float2int_rn((float)(int)(i8)(w >> (8 * i)) * ratio) & 255) << (8 * i);
    return o;
}

// One CTA writes one head of one block of one sequence, keys (blockIdx.y 0) or values (1). The new tokens stay in
// registers between the block's largest magnitude and their quantization, so they are read once; values are turned into
// rows of tokens through shared memory. The block's older tokens are touched only when its scale grows. A CTA passes through a
// chain of dependent loads (start, tokens and page, positions, tables), so what counts is how many are under way: six CTAs of
// 128 threads to an SM (4 x 8192 tokens of 8 heads of 128, F16 with rotary: 67 us, 3.0 TB/s; four of them 97 us, four of 256 threads 70 us).
// Their 80 registers do not hold the turned keys of the wider heads: at head widths 80 and 96 a thread stores 248 (F16) or 380 bytes
// (BF16) to local memory, at 128 500 or 736, and loads somewhat more; up to 64 at most 16.
template <int DT, int D>
__global__ void __launch_bounds__(128, 6) k_kv8_append(tcq_kv8_cache cache, const u16* __restrict__ k, i64 k_sb, i64 k_st,
                                                    const u16* __restrict__ v, i64 v_sb, i64 v_st, const int* __restrict__ table,
                                                    int blocks, const int* __restrict__ start, const int* __restrict__ count, RopeArgs r,
                                                    int B, int T, int NB) {
    __shared__ __align__(16) u32 tile[D * 16];
    constexpr int TH = 128;
    __shared__ u32 red[TH / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int Hk = cache.kv_heads, h = blockIdx.x % Hk, bn = blockIdx.x / Hk, n = bn % NB, b = bn / NB;
    const bool is_v = blockIdx.y != 0;
    int st = start[b], cnt = count ? count[b] : T;
    if (st < 0 || cnt < 0 || cnt > T) {
        if (threadIdx.x == 0) atomicOr(&g_tcq_memory_error, 2);
        st = max(st, 0), cnt = min(max(cnt, 0), T);
    }
    const int blk = st / kBlk + n, base = blk * kBlk;
    const int lo = max(st - base, 0), hi = min(st + cnt - base, kBlk);       // new slots of the block
    if (lo >= hi) return;
    const int page = blk < blocks ? table[(i64)b * blocks + blk] : -1;       // looked at once the tokens are on their way
    i64 off = 0;
    float* scale = nullptr;
    float s_old = 0.f;
    auto open_page = [&]() -> bool {
        if ((unsigned)page >= (unsigned)cache.pages) {
            if (threadIdx.x == 0) atomicOr(&g_tcq_memory_error, 2);
            return false;
        }
        off = ((i64)page * Hk + h) * (kBlk * D);
        scale = (is_v ? cache.v_scale : cache.k_scale) + (i64)page * Hk + h;
        if (lo > 0) s_old = *scale;
        return true;
    };
    float s, inv, ratio;
    bool grown;
    bool odd = false;
    // the block's scale from this thread's largest magnitude (as FP32 bits); finite() is that of its finite values, asked for
    // when the block holds others
    auto settle = [&](u32 top, auto finite) {
        for (;;) {
            top = __reduce_max_sync(0xffffffffu, top);
            if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < TH / 32; ++w) top = max(top, red[w]);
            if (top < 0x7f800000u) break;
            odd = true;
            top = __float_as_uint(finite());
            __syncthreads();
        }
        s = fmaxf(s_old, __uint_as_float(top) / 127.f);
        if (s < 7.52316385e-37f) s = 0.f;                         // 2^-120
        inv = s > 0.f ? 1.f / s : 0.f, ratio = s_old * inv;
        grown = lo > 0 && s > s_old;
        if (threadIdx.x == 0) *scale = s;
    };
    auto largest = [](float m, float x) {
        const float a = fabsf(x);
        return fmaxf(m, a <= 3.402823466e38f ? a : 0.f);
    };
    if (!is_v) {
        // units of 8 elements and their 8 partners of a turn: C per token, all of a thread's requested at once
        constexpr int C = D / 16, NU = (kBlk * C + TH - 1) / TH;
        const u16* src = k + b * k_sb + h * D;
        uint4 raw[NU][2];
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = threadIdx.x + TH * i, slot = u / C, c = u - slot * C;
            raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
            if (slot >= lo && slot < hi) {
                const u16* p = src + (i64)(base + slot - st) * k_st + 8 * c;
                raw[i][0] = *reinterpret_cast<const uint4*>(p), raw[i][1] = *reinterpret_cast<const uint4*>(p + D / 2);
            }
        }
        if (!open_page()) return;
        u32 top = 0;
        float x[NU][16];
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = threadIdx.x + TH * i, slot = u / C, c = u - slot * C;
            Vec<DT, 8>::unpack(raw[i][0], x[i]);
            Vec<DT, 8>::unpack(raw[i][1], x[i] + 8);
            if (r.cos_t && slot >= lo && slot < hi) {
                float cs[8], sn[8];
                rope_cs<8>(r, (i64)b * T + base + slot - st, 8 * c, cs, sn, &g_tcq_memory_error);
#pragma unroll
                for (int j = 0; j < 8; ++j) turn(x[i][j], x[i][8 + j], cs[j], sn[j]);
            }
            if (r.cos_t) {
#pragma unroll
                for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(x[i][j]) & 0x7fffffffu);
            } else {
                top = max(top, max2_bits<DT>(max2(max2(0u, raw[i][0]), raw[i][1])));
            }
        }
        settle(top, [&] {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) m = largest(m, x[i][j]);
            return m;
        });
        if (odd) {
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) x[i][j] = tamed(x[i][j], s);
        }
        i8* dst = cache.k + off;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = threadIdx.x + TH * i, slot = u / C, c = u - slot * C;
            if (slot < lo || slot >= hi) continue;
            uint2* p = reinterpret_cast<uint2*>(dst + slot * D + 8 * c);
            p[0] = make_uint2(q8x4(x[i], inv), q8x4(x[i] + 4, inv));
            p[D / 16] = make_uint2(q8x4(x[i] + 8, inv), q8x4(x[i] + 12, inv));
        }
        if (grown)
            for (int i = threadIdx.x; i < lo * (D / 4); i += TH) {
                u32* p = reinterpret_cast<u32*>(dst) + i;
                *p = requant4(*p, ratio);
            }
        return;
    }
    // values: units of 4 tokens x 8 elements, so that four tokens of an element are one word of its row. The words meet in
    // shared memory, word g of row d at g ^ (d / 8 mod 16): a warp's stores spread over the banks, and a 16-byte piece of a row
    // keeps its four words, permuted.
    constexpr int C = D / 8, NU = (16 * C + TH - 1) / TH;
    const u16* src = v + b * v_sb + h * D;
    uint4 raw[NU][4];
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        const int u = threadIdx.x + TH * i, g = u / C, c = u - g * C;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int slot = 4 * g + e;
            raw[i][e] = slot >= lo && slot < hi ? *reinterpret_cast<const uint4*>(src + (i64)(base + slot - st) * v_st + 8 * c) : make_uint4(0, 0, 0, 0);
        }
    }
    if (!open_page()) return;
    u32 top = 0;
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max2(top, raw[i][e]);
    settle(max2_bits<DT>(top), [&] {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x[8];
                Vec<DT, 8>::unpack(raw[i][e], x);
#pragma unroll
                for (int j = 0; j < 8; ++j) m = largest(m, x[j]);
            }
        return m;
    });
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        const int u = threadIdx.x + TH * i, g = u / C, c = u - g * C;
        if (16 * C % TH != 0 && u >= 16 * C) break;
        float x[4][8];
#pragma unroll
        for (int e = 0; e < 4; ++e) Vec<DT, 8>::unpack(raw[i][e], x[e]);
        if (odd) {
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j >> 3][j & 7] = tamed(x[j >> 3][j & 7], s);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float y[4] = {x[0][j], x[1][j], x[2][j], x[3][j]};
            tile[(8 * c + j) * 16 + (g ^ (c & 15))] = q8x4(y, inv);
        }
    }
    __syncthreads();
    i8* dst = cache.v + off;
#pragma unroll
    for (int i = threadIdx.x; i < D * 4; i += TH) {          // 16-token pieces of the rows
        const int d = i >> 2, t0 = (i & 3) * 16, c = (d >> 3) & 15;
        const bool any_new = t0 < hi && t0 + 16 > lo, any_old = grown && t0 < lo;
        if (!any_new && !any_old) continue;
        const uint4 f = reinterpret_cast<const uint4*>(tile)[d * 4 + ((i & 3) ^ (c >> 2))];
        const bool x1 = c & 1, x2 = c & 2;
        const u32 a0 = x1 ? f.y : f.x, a1 = x1 ? f.x : f.y, a2 = x1 ? f.w : f.z, a3 = x1 ? f.z : f.w;
        const u32 fresh[4] = {x2 ? a2 : a0, x2 ? a3 : a1, x2 ? a0 : a2, x2 ? a1 : a3};
        uint4* p = reinterpret_cast<uint4*>(dst + d * kBlk + t0);
        if (t0 >= lo && t0 + 16 <= hi) {
            *p = make_uint4(fresh[0], fresh[1], fresh[2], fresh[3]);
            continue;
        }
        const uint4 o = *p;
        u32 w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t = t0 + 4 * j;
            const u32 q = any_old ? requant4(w[j], ratio) : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u32 m = 255u << (8 * e);
                if (any_old && t + e < lo) w[j] = (w[j] & ~m) | (q & m);
                if (t + e >= lo && t + e < hi) w[j] = (w[j] & ~m) | (fresh[j] & m);
            }
        }
        *p = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ------------------------------------------------------------------------------------------------ cache read
// One CTA reads one head of one block, keys or values, and writes its tokens' rows. Values go through shared memory to
// turn rows of tokens back into tokens. Bound by HBM.
template <int DT, int D>
__global__ void __launch_bounds__(128) k_kv8_read(tcq_kv8_cache cache, char* __restrict__ ko, char* __restrict__ vo,
                                                  const int* __restrict__ table, int blocks, const int* __restrict__ begin,
                                                  const int* __restrict__ lens, int T, int NB) {
    constexpr int E = DT == TCQ_DT_F32 ? 4 : 2;
    __shared__ __align__(16) u32 tile[D * 16];
    pdl_launch_dependents();
    pdl_wait();
    const int Hk = cache.kv_heads, h = blockIdx.x % Hk, bn = blockIdx.x / Hk, n = bn % NB, b = bn / NB;
    const bool is_v = blockIdx.y != 0;
    int from = begin[b], len = lens[b];
    if (from < 0 || len < 0 || (i64)len > (i64)blocks * kBlk) {
        if (threadIdx.x == 0) atomicOr(&g_tcq_memory_error, 2);
        from = max(from, 0), len = (int)min((i64)max(len, 0), (i64)blocks * kBlk);
    }
    const i64 blk = from / kBlk + n, base = blk * kBlk;
    const int lo = (int)max((i64)from - base, (i64)0), hi = (int)min((i64)from + T - base, (i64)kBlk);
    if (lo >= hi) return;
    const int end = (int)min(max((i64)len - base, (i64)0), (i64)kBlk);        // slots that hold tokens
    int page = 0;
    if (end > lo) {
        page = table[(i64)b * blocks + blk];
        if ((unsigned)page >= (unsigned)cache.pages) {
            if (threadIdx.x == 0) atomicOr(&g_tcq_memory_error, 2);
            page = page < 0 ? 0 : cache.pages - 1;
        }
    }
    const i64 off = ((i64)page * Hk + h) * (kBlk * D);
    const float s = end > lo ? (is_v ? cache.v_scale : cache.k_scale)[(i64)page * Hk + h] : 0.f;
    char* out = (is_v ? vo : ko) + (((i64)b * T + base - from) * Hk + h) * D * E;
    const i64 row = (i64)Hk * D * E;
    auto put = [&](int slot, int d, const float* y) {             // 8 elements of a token's row
        char* o = out + slot * row + d * E;
        if (DT == TCQ_DT_F32) {
            Vec<DT, 4>::store(o, y);
            Vec<DT, 4>::store(o + 16, y + 4);
        } else {
            Vec<DT, DT == TCQ_DT_F32 ? 4 : 8>::store(o, y);
        }
    };
    if (!is_v) {
        constexpr int C = D / 8, NU = (kBlk * C + 127) / 128;
        uint2 q[NU];
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = threadIdx.x + 128 * i, slot = u / C, c = u - slot * C;
            q[i] = slot >= lo && slot < end ? *reinterpret_cast<const uint2*>(cache.k + off + slot * D + 8 * c) : make_uint2(0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = threadIdx.x + 128 * i, slot = u / C, c = u - slot * C;
            if (slot < lo || slot >= hi) continue;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = (float)(int)(i8)((j < 4 ? q[i].x : q[i].y) >> (8 * (j & 3))) * s;
            put(slot, 8 * c, y);
        }
        return;
    }
    // values: the rows of tokens through shared memory (words as in the append), then 4 tokens x 8 elements a thread
    constexpr int C = D / 8, NP = D * 4 / 128, NU = (16 * C + 127) / 128;
    if (end > lo) {
        const uint4* src = reinterpret_cast<const uint4*>(cache.v + off);
        uint4 q[NP + 1];
#pragma unroll
        for (int i = 0; i < NP + 1; ++i) {
            const int u = threadIdx.x + 128 * i;
            if (u < D * 4) q[i] = src[u];
        }
#pragma unroll
        for (int i = 0; i < NP + 1; ++i) {
            const int u = threadIdx.x + 128 * i, d = u >> 2, c = (d >> 3) & 15;
            if (u >= D * 4) break;
            const bool x1 = c & 1, x2 = c & 2;
            const u32 a0 = x1 ? q[i].y : q[i].x, a1 = x1 ? q[i].x : q[i].y, a2 = x1 ? q[i].w : q[i].z, a3 = x1 ? q[i].z : q[i].w;
            reinterpret_cast<uint4*>(tile)[d * 4 + ((u & 3) ^ (c >> 2))] = x2 ? make_uint4(a2, a3, a0, a1) : make_uint4(a0, a1, a2, a3);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        const int u = threadIdx.x + 128 * i, g = u / C, c = u - g * C;
        if (16 * C % 128 != 0 && u >= 16 * C) break;
        if (4 * g >= hi || 4 * g + 4 <= lo) continue;
        u32 w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = tile[(8 * c + j) * 16 + (g ^ (c & 15))];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int slot = 4 * g + e;
            if (slot < lo || slot >= hi) continue;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = slot < end ? (float)(int)(i8)(w[j] >> (8 * e)) * s : 0.f;
            put(slot, 8 * c, y);
        }
    }
}

}  // namespace

extern "C" {

int tcq_rope_axes(const void* x, int dtype, int64_t x_sb, int64_t x_st, void* out, int64_t o_sb, int64_t o_st, const int32_t* pos,
                  const tcq_rope_plan* plan, int B, int T, int heads, int inverse, void* stream) {
    if (!x || !out || !pos || !plan) return TCQ_ERR_ARG;
    if (dtype != TCQ_DT_BF16 && dtype != TCQ_DT_F16 && dtype != TCQ_DT_F32) return TCQ_ERR_DTYPE;
    const int e = check_rope_plan(plan);
    if (e) return e;
    if (B < 1 || T < 1 || heads < 1) return TCQ_ERR_SHAPE;
    const int es = dtype == TCQ_DT_F32 ? 4 : 2, half = plan->head_dim / 2;
    // The widest vectors that the head width, the strides and the addresses allow.
    int V = dtype == TCQ_DT_F32 ? 4 : 8;
    const uintptr_t mix = (uintptr_t)x | (uintptr_t)out | (uintptr_t)((x_sb | x_st | o_sb | o_st) * es);
    while (V > 1 && ((half % V) || (mix & (V * es - 1)))) V >>= 1;
    if (mix & (es - 1)) return TCQ_ERR_ALIGN;
    const RopeArgs r = rope_args(plan, pos, B, T);
    const float sign = inverse ? -1.f : 1.f;
#define TCQ_ROPE(DT, VV) launch_rope<DT, VV>(x, out, r, x_sb, x_st, o_sb, o_st, B, T, heads, plan->pairs != 0, sign, stream)
#define TCQ_ROPE16(DT) (V == 8 ? TCQ_ROPE(DT, 8) : V == 4 ? TCQ_ROPE(DT, 4) : V == 2 ? TCQ_ROPE(DT, 2) : TCQ_ROPE(DT, 1))
    if (dtype == TCQ_DT_BF16) return TCQ_ROPE16(TCQ_DT_BF16);
    if (dtype == TCQ_DT_F16) return TCQ_ROPE16(TCQ_DT_F16);
    return V == 4 ? TCQ_ROPE(TCQ_DT_F32, 4) : V == 2 ? TCQ_ROPE(TCQ_DT_F32, 2) : TCQ_ROPE(TCQ_DT_F32, 1);
#undef TCQ_ROPE16
#undef TCQ_ROPE
}

int tcq_kv8_append(const tcq_kv8_cache* cache, const void* k, int64_t k_sb, int64_t k_st, const void* v, int64_t v_sb, int64_t v_st,
                   int dtype, const int32_t* table, int blocks, const int32_t* start, const int32_t* count, const int32_t* pos,
                   const tcq_rope_plan* plan, int B, int T, void* stream) {
    const int e = check_cache(cache);
    if (e) return e;
    if (!k || !v || !table || !start || (plan && !pos)) return TCQ_ERR_ARG;
    if (dtype != TCQ_DT_BF16 && dtype != TCQ_DT_F16) return TCQ_ERR_DTYPE;
    if (B < 1 || T < 1 || blocks < 1) return TCQ_ERR_SHAPE;
    RopeArgs r = {};
    if (plan) {
        const int ep = check_rope_plan(plan);
        if (ep) return ep;
        if (plan->head_dim != cache->head_dim || plan->pairs) return TCQ_ERR_SHAPE;
        r = rope_args(plan, pos, B, T);
    }
    if (!tcq_aligned(k, 16) || !tcq_aligned(v, 16) || ((k_sb | k_st | v_sb | v_st) & 7)) return TCQ_ERR_ALIGN;
    const int NB = (int)(((i64)T + 2 * kBlk - 2) / kBlk);      // blocks that T tokens can touch
    const i64 ctas = (i64)B * NB * cache->kv_heads;
    if (ctas > 0x7fffffff) return TCQ_ERR_SHAPE;
    return by_head_dim(cache->head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_pdl(dtype == TCQ_DT_BF16 ? k_kv8_append<TCQ_DT_BF16, D> : k_kv8_append<TCQ_DT_F16, D>, dim3((unsigned)ctas, 2), 128, 0,
                          stream, *cache, (const u16*)k, (i64)k_sb, (i64)k_st, (const u16*)v, (i64)v_sb, (i64)v_st, table, blocks, start,
                          count, r, B, T, NB);
    });
}

int tcq_kv8_read(const tcq_kv8_cache* cache, void* k, void* v, int dtype, const int32_t* table, int blocks, const int32_t* begin,
                 const int32_t* lens, int B, int T, void* stream) {
    const int e = check_cache(cache);
    if (e) return e;
    if (!k || !v || !table || !begin || !lens) return TCQ_ERR_ARG;
    if (dtype != TCQ_DT_BF16 && dtype != TCQ_DT_F16 && dtype != TCQ_DT_F32) return TCQ_ERR_DTYPE;
    if (B < 1 || T < 1 || blocks < 1) return TCQ_ERR_SHAPE;
    if (!tcq_aligned(k, 16) || !tcq_aligned(v, 16)) return TCQ_ERR_ALIGN;
    const int NB = (int)(((i64)T + 2 * kBlk - 2) / kBlk);
    const i64 ctas = (i64)B * NB * cache->kv_heads;
    if (ctas > 0x7fffffff) return TCQ_ERR_SHAPE;
    return by_head_dim(cache->head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        auto kern = dtype == TCQ_DT_BF16 ? k_kv8_read<TCQ_DT_BF16, D> : dtype == TCQ_DT_F16 ? k_kv8_read<TCQ_DT_F16, D> : k_kv8_read<TCQ_DT_F32, D>;
        return launch_pdl(kern, dim3((unsigned)ctas, 2), 128, 0, stream, *cache, (char*)k, (char*)v, table, blocks, begin, lens, T, NB);
    });
}

}  // extern "C"
