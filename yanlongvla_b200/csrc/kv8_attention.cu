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

}  // namespace

extern "C" {

size_t tcq_kv8_attention_workspace(int B, int T, int heads, int kv_heads, int head_dim, int blocks) {
    if (B < 1 || T < 1 || heads < 1 || kv_heads < 1 || head_dim < 1 || blocks < 1) return 0;
    return 16;
}

int tcq_kv8_attention(const tcq_kv8_cache* cache, const void* q, int dtype, int64_t q_sb, int64_t q_st, void* out, const int32_t* table,
                      int blocks, const int32_t* lens, const int32_t* count, int causal, float scale, int B, int T, int heads,
                      void* workspace, size_t workspace_bytes, void* stream) {
    const int e = check_cache(cache);
    if (e) return e;
    if (!q || !out || !table || !lens) return TCQ_ERR_ARG;
    if (dtype != TCQ_DT_BF16 && dtype != TCQ_DT_F16) return TCQ_ERR_DTYPE;
    if (B < 1 || T < 1 || blocks < 1 || heads < 1 || heads % cache->kv_heads || blocks > (0x7fffffff / kBlk)) return TCQ_ERR_SHAPE;
    if (!tcq_aligned(q, 16) || !tcq_aligned(out, 16) || ((q_sb | q_st) & 7)) return TCQ_ERR_ALIGN;
    if (!workspace || workspace_bytes < tcq_kv8_attention_workspace(B, T, heads, cache->kv_heads, cache->head_dim, blocks))
        return TCQ_ERR_WORKSPACE;
    const i64 rows = (i64)B * T * heads;
    if ((rows + 3) / 4 > 0x7fffffff) return TCQ_ERR_SHAPE;
    return by_head_dim(cache->head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_pdl(dtype == TCQ_DT_BF16 ? k_attention_rows<TCQ_DT_BF16, D> : k_attention_rows<TCQ_DT_F16, D>,
                          dim3((unsigned)((rows + 3) / 4)), 128, 0, stream, *cache, (const u16*)q, (i64)q_sb, (i64)q_st, (u16*)out, table,
                          blocks, lens, count, causal, scale, rows, T, heads);
    });
}

}  // extern "C"
