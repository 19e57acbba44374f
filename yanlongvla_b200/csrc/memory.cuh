// Shared pieces of the streaming-memory kernels: the rotary embedding with several axes, 16-bit element types, and the
// flag that reports an index out of range.
#pragma once
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "tcq_common.cuh"

namespace tcq {

typedef long long i64;

constexpr int kBlk = TCQ_KV8_BLOCK;      // tokens of a cache block (a page)

// ---------------------------------------------------------------------------------------------------- element types
template <int DT>
TCQ_HD float elem_f(u16 b) { return DT == TCQ_DT_F16 ? h2f(b) : bf2f(b); }

// Two FP32 values as a packed pair of the type, rounded to nearest even; lo in the low half.
template <int DT>
TCQ_HD u32 pack2(float lo, float hi) {
    if (DT == TCQ_DT_F16) {
        u32 r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    return f2bf2(lo, hi);
}

template <int DT>
TCQ_HD void unpack2(u32 w, float& lo, float& hi) {
    if (DT == TCQ_DT_F16) {
        __half2 h;
        memcpy(&h, &w, 4);
        const float2 f = __half22float2(h);
        lo = f.x, hi = f.y;
    } else {
        lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u);
    }
}

// ---------------------------------------------------------------------------------------------------- rotary tables
struct RopeArgs {
    const float* cos_t;
    const float* sin_t;
    const int* pos;          // (axes, B, T)
    i64 axis_stride;         // B * T
    int positions, half;     // table rows, frequencies of a head
    int e0, e1, e2;          // first frequency of axes 1, 2, 3
};

static inline RopeArgs rope_args(const tcq_rope_plan* p, const int32_t* pos, int B, int T) {
    RopeArgs r;
    r.cos_t = p->cos_t;
    r.sin_t = p->sin_t;
    r.pos = pos;
    r.axis_stride = (i64)B * T;
    r.positions = p->positions;
    r.half = p->head_dim / 2;
    r.e0 = p->section[0];
    r.e1 = r.e0 + p->section[1];
    r.e2 = r.e1 + p->section[2];
    if (p->axes < 2) r.e0 = 1 << 30;
    if (p->axes < 3) r.e1 = 1 << 30;
    if (p->axes < 4) r.e2 = 1 << 30;
    return r;
}

static inline int check_rope_plan(const tcq_rope_plan* p) {
    if (!p->cos_t || !p->sin_t) return TCQ_ERR_ARG;
    if (p->axes < 1 || p->axes > 4 || p->positions < 1 || p->head_dim < 2 || p->head_dim > 256 || (p->head_dim & 1)) return TCQ_ERR_SHAPE;
    int sum = 0;
    for (int a = 0; a < p->axes; ++a) {
        if (p->section[a] < 0) return TCQ_ERR_SHAPE;
        sum += p->section[a];
    }
    if (sum != p->head_dim / 2) return TCQ_ERR_SHAPE;
    return tcq_aligned(p->cos_t, 16) && tcq_aligned(p->sin_t, 16) ? TCQ_OK : TCQ_ERR_ALIGN;
}

// Cosines and sines of frequencies j0 .. j0 + V - 1 of token `row` = b * T + t (V 1, 2, 4 or 8; j0 a multiple of V). Four
// frequencies of one axis are one 16-byte load of each table (rows of half * 4 bytes: aligned when half is a multiple of 4).
template <int V>
TCQ_HD void rope_cs(const RopeArgs& r, i64 row, int j0, float* c, float* s, int* err) {
    auto at = [&](int j) -> i64 {
        const int a = (j >= r.e0) + (j >= r.e1) + (j >= r.e2);
        int p = __ldg(r.pos + a * r.axis_stride + row);
        if ((unsigned)p >= (unsigned)r.positions) {
            atomicOr(err, 2);
            p = p < 0 ? 0 : r.positions - 1;
        }
        return (i64)p * r.half + j;
    };
    constexpr int G = V >= 4 ? V / 4 : 1, W = V >= 4 ? 4 : V;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const int j = j0 + 4 * g;
        const bool one = W == 4 && (r.half & 3) == 0 &&
                         ((j >= r.e0) == (j + 3 >= r.e0)) && ((j >= r.e1) == (j + 3 >= r.e1)) && ((j >= r.e2) == (j + 3 >= r.e2));
        if (one) {
            const i64 o = at(j);
            const float4 c4 = __ldg(reinterpret_cast<const float4*>(r.cos_t + o)), s4 = __ldg(reinterpret_cast<const float4*>(r.sin_t + o));
            c[4 * g] = c4.x, c[4 * g + 1] = c4.y, c[4 * g + 2] = c4.z, c[4 * g + 3] = c4.w;
            s[4 * g] = s4.x, s[4 * g + 1] = s4.y, s[4 * g + 2] = s4.z, s[4 * g + 3] = s4.w;
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const i64 o = at(j + i);
                c[4 * g + i] = __ldg(r.cos_t + o);
                s[4 * g + i] = __ldg(r.sin_t + o);
            }
        }
    }
}

// (a, b) -> (a c - b s, a s + b c), one rounding per operation.
TCQ_HD void turn(float& a, float& b, float c, float s) {
    const float p = a * c, q = b * s, u = a * s, v = b * c;
    a = p - q;
    b = u + v;
}

// ---------------------------------------------------------------------------------------------------- host helpers
// Launch with programmatic dependent launch, as every kernel of the library.
template <class... P, class... A>
static inline int launch_pdl(void (*kern)(P...), dim3 grid, int threads, size_t smem, void* stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, P(args)...) == cudaSuccess ? TCQ_OK : TCQ_ERR_LAUNCH;
}

// The same for a kernel with more than 48 KB of dynamic shared memory; the attribute is set once per device.
template <auto Kern, class... A>
static inline int launch_big(dim3 grid, int threads, size_t smem, void* stream, const A&... args) {
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return TCQ_ERR_DEVICE;
    if (!(set.load(std::memory_order_relaxed) >> dev & 1)) {
        if (cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return TCQ_ERR_LAUNCH;
        set.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return launch_pdl(Kern, grid, threads, smem, stream, args...);
}

static inline int check_cache(const tcq_kv8_cache* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return TCQ_ERR_ARG;
    if (c->pages < 1 || c->kv_heads < 1) return TCQ_ERR_SHAPE;
    switch (c->head_dim) {
        case 32: case 48: case 64: case 80: case 96: case 128: break;
        default: return TCQ_ERR_SHAPE;
    }
    return tcq_aligned(c->k, 16) && tcq_aligned(c->v, 16) ? TCQ_OK : TCQ_ERR_ALIGN;
}

// Call f(integral_constant<int, D>) for the head width.
template <class F>
static inline int by_head_dim(int d, F f) {
    switch (d) {
        case 32: return f(std::integral_constant<int, 32>());
        case 48: return f(std::integral_constant<int, 48>());
        case 64: return f(std::integral_constant<int, 64>());
        case 80: return f(std::integral_constant<int, 80>());
        case 96: return f(std::integral_constant<int, 96>());
        default: return f(std::integral_constant<int, 128>());
    }
}

}  // namespace tcq
