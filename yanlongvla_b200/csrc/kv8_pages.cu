// Pages of the 8-bit cache: sequences that share pages (fork), pages for new tokens (reserve), copies of pages, tokens packed
// into other pages (compact), pages given back (free).
//
// refs[p] counts the table entries that name page p; 0 is a free page. A row of a table names its sequence's pages from block 0 on
// and -1 behind them. The book-keeping kernels are bound by the chain of their dependent loads (0.6 to 0.8 us each), the copies by HBM.
#include "memory.cuh"

__device__ int g_tcq_pages_error;

int tcq_pages_error(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tcq_pages_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && v) {
        const int z = 0;
        if (cudaMemcpyToSymbol(g_tcq_pages_error, &z, sizeof(int)) != cudaSuccess) return -1;
    }
    return v;
}

namespace {

using namespace tcq;

TCQ_HD void out_of_range() { atomicOr(&g_tcq_pages_error, 2); }

TCQ_HD int clamped(int n, int lo, int hi) {
    if (n < lo || n > hi) {
        out_of_range();
        return n < lo ? lo : hi;
    }
    return n;
}
TCQ_HD int blocks_of(int tokens) { return tokens / kBlk + (tokens % kBlk != 0); }

// ------------------------------------------------------------------------------------------------ fork
// Row b becomes what row parent[b] was, all rows at once. A cluster of eight CTAs takes the table's columns, C at a time: a tile of
// all rows is staged in shared memory, so that rows may change places in the table itself. Lengths are read by every CTA before
// the cluster's barrier and written by one behind it.
constexpr int kForkCtas = 8, kForkThreads = 512, kForkTile = 64 * 1024;

__global__ void __launch_bounds__(kForkThreads, 1) k_kv8_fork(int* __restrict__ refs, int pages, int* __restrict__ table, int blocks,
                                                              int* __restrict__ lens, const int* __restrict__ parent, int B, int shift) {
    extern __shared__ int s_mem[];
    int *s_from = s_mem, *s_len = s_mem + B, *s_tile = s_mem + 2 * B;      // parent, tokens of the row's old sequence, a tile
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, C = 1 << shift, rank = blockIdx.x;
    for (int b = tid; b < B; b += kForkThreads) {
        int p = parent[b];
        if (p >= B) {
            out_of_range();
            p = b;
        }
        s_from[b] = p;
        s_len[b] = clamped(lens[b], 0, (int)min((i64)blocks * kBlk, (i64)0x7fffffff));
    }
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
#pragma unroll 1
    for (int c0 = rank * C; c0 < blocks; c0 += kForkCtas * C) {
        const int n = B << shift;
#pragma unroll 8
        for (int i = tid; i < n; i += kForkThreads) {
            const int b = i >> shift, c = c0 + (i & (C - 1));
            s_tile[i] = c < blocks ? table[(i64)b * blocks + c] : -1;
        }
        __syncthreads();
        for (int i = tid; i < n; i += kForkThreads) {
            const int b = i >> shift, c = c0 + (i & (C - 1)), p = s_from[b];
            if (p == b || c >= blocks) continue;
            const int old = s_tile[i];
            int now = p < 0 || c >= blocks_of(s_len[p]) ? -1 : s_tile[(p << shift) + (i & (C - 1))];
            if (now >= pages) {
                out_of_range();
                now = -1;
            }
            if (old >= 0 && old < pages) atomicAdd(refs + old, -1);
            if (now >= 0) atomicAdd(refs + now, 1);
            if (now != old) table[(i64)b * blocks + c] = now < 0 ? -1 : now;
        }
        __syncthreads();
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0)
        for (int b = tid; b < B; b += kForkThreads) lens[b] = s_from[b] < 0 ? 0 : s_len[s_from[b]];
}

// ------------------------------------------------------------------------------------------------ free
// A thread for each entry of the table. lens[b] may be read before or after its own thread has lowered it: min(keep, lens) is the
// same.
__global__ void __launch_bounds__(256) k_kv8_free(int* __restrict__ refs, int pages, int* __restrict__ table, int blocks, int* lens,
                                                  const int* __restrict__ keep, int B) {
    pdl_launch_dependents();
    pdl_wait();
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), b = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (b >= B) return;
    const i64 at = (i64)b * blocks + c;
    const int p = c < blocks ? table[at] : -1;
    const int len = *(volatile int*)(lens + b), hold = max(min(keep[b], len), 0);
    if (c == 0 && keep[b] < 0) out_of_range();
    if (p >= 0 && c >= blocks_of(hold)) {
        if (p < pages) atomicAdd(refs + p, -1);
        table[at] = -1;
    }
    if (c == 0 && len != hold) lens[b] = hold;
}

// ------------------------------------------------------------------------------------------------ reserve
// One CTA, since the pages go out in order. Of sequence b the blocks first .. last - 1 get tokens; its missing pages are those of the
// trailing -1 entries among them, before them a page for the begun block where others share it. A scan of those numbers says which
// sequences fit; a scan of the free pages, 16 of a thread at a time, gives the r-th free page to the sequence that holds number
// r. The first 16384 pages are requested with the lengths, so that a small pool costs no further load.
constexpr int kResThreads = 1024, kResPer = 16, kResChunk = kResThreads * kResPer;

// Exclusive sum of v over the CTA; all: the sum.
TCQ_HD int block_scan(int v, int* s_warp, int& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int scan = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += u;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = scan;
    __syncthreads();
    int w = s_warp[lane], before = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
    }
    all = __shfl_sync(0xffffffffu, before, 31);
    return scan - v + __shfl_sync(0xffffffffu, before - w, warp);
}

// Bit i: page base + i is free.
TCQ_HD u32 free_mask(const int* refs, int pages, i64 base) {
    u32 m = 0;
    if (base + kResPer <= pages && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) {
        int4 v[kResPer / 4];
#pragma unroll
        for (int i = 0; i < kResPer / 4; ++i) v[i] = __ldcg(reinterpret_cast<const int4*>(refs + base) + i);
#pragma unroll
        for (int i = 0; i < kResPer / 4; ++i)
            m |= (u32)(v[i].x == 0) << (4 * i) | (u32)(v[i].y == 0) << (4 * i + 1) | (u32)(v[i].z == 0) << (4 * i + 2) | (u32)(v[i].w == 0) << (4 * i + 3);
    } else {
        for (int i = 0; i < kResPer; ++i)
            if (base + i < pages && __ldcg(refs + base + i) == 0) m |= 1u << i;
    }
    return m;
}

__global__ void __launch_bounds__(kResThreads, 1) k_kv8_reserve(int* refs, int pages, int* __restrict__ table, int blocks,
                                                                const int* __restrict__ lens, const int* __restrict__ count,
                                                                int* __restrict__ granted, int* __restrict__ copies, int B, int lanes) {
    extern __shared__ int s_mem[];
    int *s_upto = s_mem, *s_first = s_mem + B, *s_begun = s_mem + 2 * B;   // missing pages up to a sequence, first missing block, begun page
    __shared__ int s_warp[32];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, sub = tid & (lanes - 1), per_pass = kResThreads / lanes;
    const int limit = (int)min((i64)blocks * kBlk, (i64)0x7fffffff);
    const u32 mask0 = free_mask(refs, pages, (i64)tid * kResPer);
    for (int b0 = 0; b0 < B; b0 += per_pass) {
        const int b = b0 + tid / lanes;
        int missing = 0, first = 0, last = 0, at = -1, cnt = 0;
        bool fits = true;
        if (b < B) {
            const int len = clamped(lens[b], 0, limit);
            cnt = count[b];
            if (cnt < 0) out_of_range();
            fits = cnt <= limit - len;
            if (cnt > 0 && fits) {
                first = len / kBlk, last = blocks_of(len + cnt);
                const bool begun = len % kBlk != 0;
                if (begun) {
                    at = table[(i64)b * blocks + first];
                    if ((unsigned)at >= (unsigned)pages) fits = false, at = -1;
                }
                for (int j = first + begun + sub; j < last; j += lanes) missing += table[(i64)b * blocks + j] < 0;
            }
        }
        for (int o = 1; o < lanes; o <<= 1) missing += __shfl_xor_sync(0xffffffffu, missing, o);
        if (b < B && sub == 0) {
            if (!fits) out_of_range();
            const bool want = cnt > 0 && fits;
            s_upto[b] = want ? missing : -1;                                // -1: nothing asked for, or no room in the table
            s_first[b] = want ? last - missing : 0;
            s_begun[b] = want && at >= 0 && __ldcg(refs + at) > 1 ? at : -1;
        }
    }
    __syncthreads();
    // Writers of shared pages let them go; where that leaves none, the last of them (the highest number) keeps the page.
    for (int b = tid; b < B; b += kResThreads)
        if (s_begun[b] >= 0) atomicAdd(refs + s_begun[b], -1);
    __syncthreads();
    for (int b0 = 0; b0 < B; b0 += kResThreads) {
        const int b = b0 + tid;
        if (b < B && s_begun[b] >= 0 && __ldcg(refs + s_begun[b]) <= 0) s_begun[b] |= 1 << 30;
    }
    __syncthreads();
    for (int b = tid; b < B; b += kResThreads)
        if (s_begun[b] >= 0 && s_begun[b] >> 30) atomicMax(refs + (s_begun[b] & ~(1 << 30)), b + 1);
    __syncthreads();
    for (int b = tid; b < B; b += kResThreads) {
        const int at = s_begun[b];
        if (at >= 0 && at >> 30) s_begun[b] = __ldcg(refs + (at & ~(1 << 30))) == b + 1 ? -2 - (at & ~(1 << 30)) : at & ~(1 << 30);
    }
    __syncthreads();
    for (int b = tid; b < B; b += kResThreads)
        if (s_begun[b] <= -2) {
            refs[-2 - s_begun[b]] = 1;
            s_begun[b] = -1;
        }
    __syncthreads();
    // sequences in order, a run of them to a thread: missing pages up to and with each
    const int run = (B + kResThreads - 1) / kResThreads, r0 = min(B, tid * run), r1 = min(B, r0 + run);
    int mine = 0, all;
    for (int b = r0; b < r1; ++b) mine += max(s_upto[b], 0) + (s_begun[b] >= 0);
    int upto = block_scan(mine, s_warp, all);
    // free pages, until there are enough
    int found = 0;
    const int chunks = (pages + kResChunk - 1) / kResChunk;
    for (int ch = 0; ch < chunks && found < all; ++ch) {
        const u32 m = ch == 0 ? mask0 : free_mask(refs, pages, (i64)ch * kResChunk + tid * kResPer);
        int n;
        block_scan(__popc(m), s_warp, n);
        found += n;
    }
    int refused = 0;
    for (int b = r0; b < r1; ++b) {
        const bool asked = s_upto[b] >= 0, copied = s_begun[b] >= 0;
        upto += max(s_upto[b], 0) + copied;
        const bool ok = asked && upto <= found;
        granted[b] = ok ? count[b] : 0;
        if (!(ok && copied)) copies[b] = copies[B + b] = -1;
        else copies[b] = s_begun[b];
        if (asked && !ok) {
            refused = 1;
            if (copied) atomicAdd(refs + s_begun[b], 1);
        }
        s_upto[b] = upto;
    }
    if (refused) out_of_range();
    __syncthreads();
    // The pages of number 0 .. take - 1 go out: what the last sequence that fits needs, found by bisection.
    auto sequence_of = [&](int r) -> int {                                  // the first with s_upto > r
        int lo = 0, hi = B - 1;
        while (lo < hi) {
            const int m = (lo + hi) >> 1;
            if (s_upto[m] > r) hi = m;
            else lo = m + 1;
        }
        return lo;
    };
    int take = all;
    if (found < all) {
        const int b = sequence_of(found);                                   // the first that does not fit
        take = b > 0 ? s_upto[b - 1] : 0;
    }
    int given = 0;
    for (int ch = 0; ch < chunks && given < take; ++ch) {
        u32 m = ch == 0 ? mask0 : free_mask(refs, pages, (i64)ch * kResChunk + tid * kResPer);
        int n, r = block_scan(__popc(m), s_warp, n) + given;
        given += n;
        for (; m && r < take; m &= m - 1, ++r) {
            const int page = ch * kResChunk + tid * kResPer + __ffs(m) - 1, b = sequence_of(r);
            const int k = r - (b > 0 ? s_upto[b - 1] : 0);
            int j = s_first[b] + k;
            if (s_begun[b] >= 0) {
                j = k == 0 ? min(max(lens[b], 0), limit) / kBlk : j - 1;
                if (k == 0) copies[B + b] = page;
            }
            refs[page] = 1;
            table[(i64)b * blocks + j] = page;
        }
    }
}

// ------------------------------------------------------------------------------------------------ copies of pages
struct Layers {
    struct {
        i8 *k, *v;
        float *ks, *vs;
    } at[TCQ_KV8_MAX_LAYERS];
};

// A CTA moves 32 KB of one page's keys (blockIdx.z even) or values, eight 16-byte loads of a thread under way.
__global__ void __launch_bounds__(256) k_kv8_copy(const __grid_constant__ Layers L, const int* __restrict__ copies, int n, int pages, int heads, int cells) {
    pdl_launch_dependents();
    pdl_wait();
    const int src = copies[blockIdx.x], dst = copies[n + blockIdx.x], tid = threadIdx.x;
    if (src < 0 || dst < 0 || src == dst) return;
    if (src >= pages || dst >= pages) {
        if (tid == 0) out_of_range();
        return;
    }
    const bool is_v = blockIdx.z & 1;
    const auto& l = L.at[blockIdx.y];
    const i64 page = (i64)heads * cells;                                    // bytes
    i8* const base = is_v ? l.v : l.k;
    const uint4* s = reinterpret_cast<const uint4*>(base + src * page);
    uint4* d = reinterpret_cast<uint4*>(base + dst * page);
    const int words = (int)(page / 16), i0 = (blockIdx.z >> 1) * 2048;
    uint4 w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i0 + i * 256 + tid < words) w[i] = s[i0 + i * 256 + tid];
    if (i0 == 0) {
        float* sc = is_v ? l.vs : l.ks;
        for (int h = tid; h < heads; h += 256) sc[(i64)dst * heads + h] = sc[(i64)src * heads + h];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i0 + i * 256 + tid < words) d[i0 + i * 256 + tid] = w[i];
}

// ------------------------------------------------------------------------------------------------ compact
// A CTA writes one head of one block of new pages, keys (blockIdx.z even) or values, in one layer: for its up to 64 tokens the page
// and slot they come from, s = the largest of their pages' scales, q' = rint(q (s_old / s)) (a token whose page has that scale
// keeps its integers). Keys are rows of a token: 16 bytes of one a thread. Values lie token by token along a row, so the source
// pages' tiles pass through shared memory, from which four tokens' bytes make a word.
//
// Quotients of integers q' = q r with 0 <= r <= 1: the byte in a float's low bits (2^23 + 128 + q), its offset taken off, times r,
// rounded to nearest even by adding 1.5 * 2^23.
TCQ_HD u32 scaled4(u32 w, const float (&r)[4]) {
    const u32 u = w ^ 0x80808080u;
    u32 b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint((__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + i)) - 8388736.f) * r[i] + 12582912.f);
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

template <int D>
__global__ void __launch_bounds__(128) k_kv8_compact(const __grid_constant__ Layers L, const int* __restrict__ table, int blocks,
                                                     const int* __restrict__ lens, const int* __restrict__ index, int M,
                                                     const int* __restrict__ kept, const int* __restrict__ new_table, int new_blocks,
                                                     int pages, int heads, int NB) {
    constexpr int TH = 128, PAGE = kBlk * D;
    __shared__ __align__(16) char tile[2 * PAGE];          // up to two source pages' values
    __shared__ int s_page[kBlk], s_slot[kBlk];
    __shared__ float s_ratio[kBlk];
    __shared__ float s_top[2];
    pdl_launch_dependents();
    pdl_wait();
    const int h = blockIdx.x % heads, bn = blockIdx.x / heads, n = bn % NB, b = bn / NB, tid = threadIdx.x;
    const bool is_v = blockIdx.z & 1;
    const auto& l = L.at[blockIdx.y];
    int m = M;
    if (kept) {
        m = kept[b];
        if (m < 0 || m > M) {
            if (tid == 0) out_of_range();
            m = m < 0 ? 0 : M;
        }
    }
    const int live = min(m - n * kBlk, kBlk);
    if (live <= 0) return;
    const int to = n < new_blocks ? new_table[(i64)b * new_blocks + n] : -1;
    if ((unsigned)to >= (unsigned)pages) {
        if (tid == 0) out_of_range();
        return;
    }
    const float* scale = is_v ? l.vs : l.ks;
    if (tid < kBlk) {
        int page = -1, slot = 0;
        float s = 0.f;
        if (tid < live) {
            const int len = min(lens[b], (int)min((i64)blocks * kBlk, (i64)0x7fffffff));
            int i = index[(i64)b * M + n * kBlk + tid];
            bool ok = (unsigned)i < (unsigned)max(len, 0);
            if (ok) {
                slot = i % kBlk;
                page = table[(i64)b * blocks + i / kBlk];
                ok = (unsigned)page < (unsigned)pages;
            }
            if (ok) s = scale[(i64)page * heads + h];
            else page = -1, out_of_range();
        }
        float top = s;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((tid & 31) == 0) s_top[tid >> 5] = top;
        s_page[tid] = page, s_slot[tid] = slot;
        s_ratio[tid] = s;
    }
    __syncthreads();
    const float top = fmaxf(s_top[0], s_top[1]);
    if (tid < kBlk) s_ratio[tid] = top > 0.f ? s_ratio[tid] / top : 0.f;
    if (tid == 0) (is_v ? l.vs : l.ks)[(i64)to * heads + h] = top;
    const i64 dst = ((i64)to * heads + h) * PAGE;
    __syncthreads();
    if (!is_v) {
        constexpr int C = D / 16, NU = (kBlk * C + TH - 1) / TH;
        uint4 w[NU];
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = tid + TH * i, t = u / C, c = u - t * C;
            if (kBlk * C % TH != 0 && u >= kBlk * C) break;
            const int page = s_page[t];
            w[i] = page < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(l.k + ((i64)page * heads + h) * PAGE + s_slot[t] * D + 16 * c);
        }
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = tid + TH * i, t = u / C;
            if (kBlk * C % TH != 0 && u >= kBlk * C) break;
            const float r = s_ratio[t];
            if (r != 1.f) {
                const float r4[4] = {r, r, r, r};
                w[i].x = scaled4(w[i].x, r4), w[i].y = scaled4(w[i].y, r4), w[i].z = scaled4(w[i].z, r4), w[i].w = scaled4(w[i].w, r4);
            }
            *reinterpret_cast<uint4*>(l.k + dst + 16 * u) = w[i];
        }
        return;
    }
    // Values: word (d, g) holds tokens 4 g .. 4 g + 3 of element d. Sixteen lanes to a row, so that bytes of neighbouring tokens
    // come from neighbouring words.
    constexpr int NW = D * 16 / TH, ROWS = TH / 16;
    const int g = tid & 15, d0 = tid >> 4;
    u32 out[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) out[i] = 0;
    int mypage[4], myslot[4];
    float r4[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) mypage[e] = s_page[4 * g + e], myslot[e] = s_slot[4 * g + e], r4[e] = s_ratio[4 * g + e];
    // runs of tokens of one page, two at a time
    for (int t = 0; t < live;) {
        int page[2] = {-1, -1}, from[2], end = t;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            from[k] = end;
            if (end >= live) continue;
            page[k] = s_page[end];
            while (end < live && s_page[end] == page[k]) ++end;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (page[k] >= 0) {
                const char* src = reinterpret_cast<const char*>(l.v + ((i64)page[k] * heads + h) * PAGE);
#pragma unroll
                for (int i = 0; i < (PAGE / 16 + TH - 1) / TH; ++i)
                    if (PAGE / 16 % TH == 0 || tid + TH * i < PAGE / 16) cp_async16(tile + k * PAGE + (tid + TH * i) * 16, src + (tid + TH * i) * 16);
            }
        cp_async_wait_all();
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int p = 4 * g + e;
            if (p >= t && p < end && mypage[e] >= 0) {
                const char* src = tile + (p >= from[1] && page[1] >= 0 ? PAGE : 0) + myslot[e];
#pragma unroll
                for (int i = 0; i < NW; ++i) out[i] |= (u32)(unsigned char)src[(d0 + ROWS * i) * kBlk] << (8 * e);
            }
        }
        t = end;
    }
    const bool same = r4[0] == 1.f && r4[1] == 1.f && r4[2] == 1.f && r4[3] == 1.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        if (!same) out[i] = scaled4(out[i], r4);
        reinterpret_cast<u32*>(l.v + dst)[(d0 + ROWS * i) * 16 + g] = out[i];
    }
}

int check_layers(const tcq_kv8_cache* c, int layers) {
    if (!c || layers < 1) return TCQ_ERR_ARG;
    for (int i = 0; i < layers; ++i) {
        const int e = check_cache(c + i);
        if (e) return e;
        if (c[i].pages != c[0].pages || c[i].kv_heads != c[0].kv_heads || c[i].head_dim != c[0].head_dim) return TCQ_ERR_SHAPE;
    }
    return TCQ_OK;
}

// f(first layer, layers, their pointers) for up to TCQ_KV8_MAX_LAYERS layers at a time.
template <class F>
int by_layers(const tcq_kv8_cache* c, int layers, F f) {
    for (int i0 = 0; i0 < layers; i0 += TCQ_KV8_MAX_LAYERS) {
        const int n = layers - i0 < TCQ_KV8_MAX_LAYERS ? layers - i0 : TCQ_KV8_MAX_LAYERS;
        Layers L = {};
        for (int i = 0; i < n; ++i) L.at[i] = {c[i0 + i].k, c[i0 + i].v, c[i0 + i].k_scale, c[i0 + i].v_scale};
        const int e = f(n, L);
        if (e) return e;
    }
    return TCQ_OK;
}

int check_table(const void* refs, int pages, const void* table, int blocks, const void* lens, int B) {
    if (!refs || !table || !lens) return TCQ_ERR_ARG;
    return pages < 1 || blocks < 1 || B < 1 || B > TCQ_KV8_MAX_SEQUENCES || pages > (1 << 30) - 1 ? TCQ_ERR_SHAPE : TCQ_OK;
}

}  // namespace

extern "C" {

int tcq_kv8_fork(int32_t* refs, int pages, int32_t* table, int blocks, int32_t* lens, const int32_t* parent, int B, void* stream) {
    const int e = check_table(refs, pages, table, blocks, lens, B);
    if (e) return e;
    if (!parent) return TCQ_ERR_ARG;
    // columns of a tile: 32 (a line of the table), fewer where all rows' would not fit; no more than the eight CTAs share evenly
    int shift = 5;
    while (shift > 0 && ((i64)B << shift) * 4 > kForkTile) --shift;
    while (shift > 2 && blocks <= (kForkCtas << (shift - 1))) --shift;
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return TCQ_ERR_DEVICE;
    constexpr int most = kForkTile + 8 * TCQ_KV8_MAX_SEQUENCES;
    if (!(set.load(std::memory_order_relaxed) >> dev & 1)) {
        if (cudaFuncSetAttribute(k_kv8_fork, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) return TCQ_ERR_LAUNCH;
        set.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kForkCtas);
    cfg.blockDim = dim3(kForkThreads);
    cfg.dynamicSmemBytes = (size_t)4 * (((size_t)B << shift) + 2 * B);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kForkCtas, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k_kv8_fork, (int*)refs, pages, (int*)table, blocks, (int*)lens, (const int*)parent, B, shift) == cudaSuccess
               ? TCQ_OK : TCQ_ERR_LAUNCH;
}

int tcq_kv8_free(int32_t* refs, int pages, int32_t* table, int blocks, int32_t* lens, const int32_t* keep, int B, void* stream) {
    const int e = check_table(refs, pages, table, blocks, lens, B);
    if (e) return e;
    if (!keep) return TCQ_ERR_ARG;
    return launch_pdl(k_kv8_free, dim3((blocks + 31) / 32, (B + 7) / 8), 256, 0, stream, (int*)refs, pages, (int*)table, blocks, (int*)lens,
                      (const int*)keep, B);
}

int tcq_kv8_reserve(int32_t* refs, int pages, int32_t* table, int blocks, const int32_t* lens, const int32_t* count, int32_t* granted,
                    int32_t* copies, int B, void* stream) {
    const int e = check_table(refs, pages, table, blocks, lens, B);
    if (e) return e;
    if (!count || !granted || !copies) return TCQ_ERR_ARG;
    // lanes that look through a sequence's entries side by side: what 1024 threads allow
    int lanes = 32;
    while (lanes > 1 && B * lanes > kResThreads) lanes >>= 1;
    constexpr int most = 12 * TCQ_KV8_MAX_SEQUENCES;
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return TCQ_ERR_DEVICE;
    if (!(set.load(std::memory_order_relaxed) >> dev & 1)) {
        if (cudaFuncSetAttribute(k_kv8_reserve, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) return TCQ_ERR_LAUNCH;
        set.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return launch_pdl(k_kv8_reserve, dim3(1), kResThreads, (size_t)12 * B, stream, (int*)refs, pages, (int*)table, blocks, (const int*)lens,
                      (const int*)count, (int*)granted, (int*)copies, B, lanes);
}

int tcq_kv8_copy(const tcq_kv8_cache* caches, int layers, const int32_t* copies, int n, void* stream) {
    const int e = check_layers(caches, layers);
    if (e) return e;
    if (!copies) return TCQ_ERR_ARG;
    if (n < 1) return TCQ_ERR_SHAPE;
    const int cells = kBlk * caches->head_dim, heads = caches->kv_heads;
    const i64 parts = ((i64)heads * cells / 16 + 2047) / 2048;
    if (parts * 2 > 65535) return TCQ_ERR_SHAPE;
    return by_layers(caches, layers, [&](int count, const Layers& L) {
        return launch_pdl(k_kv8_copy, dim3(n, count, (unsigned)(2 * parts)), 256, 0, stream, L, (const int*)copies, n, caches->pages, heads, cells);
    });
}

int tcq_kv8_compact(const tcq_kv8_cache* caches, int layers, const int32_t* table, int blocks, const int32_t* lens, const int32_t* index,
                    int tokens, const int32_t* kept, const int32_t* new_table, int new_blocks, int B, void* stream) {
    const int e = check_layers(caches, layers);
    if (e) return e;
    if (!table || !lens || !index || !new_table) return TCQ_ERR_ARG;
    if (B < 1 || tokens < 1 || blocks < 1 || new_blocks < 1) return TCQ_ERR_SHAPE;
    const int NB = (tokens + kBlk - 1) / kBlk, heads = caches->kv_heads;
    const i64 ctas = (i64)B * NB * heads;
    if (ctas > 0x7fffffff) return TCQ_ERR_SHAPE;
    return by_layers(caches, layers, [&](int count, const Layers& L) {
        return by_head_dim(caches->head_dim, [&](auto d) {
            return launch_pdl(k_kv8_compact<decltype(d)::value>, dim3((unsigned)ctas, count, 2), 128, 0, stream, L, (const int*)table, blocks,
                              (const int*)lens, (const int*)index, tokens, (const int*)kept, (const int*)new_table, new_blocks,
                              caches->pages, heads, NB);
        });
    });
}

}  // extern "C"
