// Pages of the 8-bit cache: sequences that share pages (fork), pages for new tokens (reserve), copies of pages, tokens packed
// into other pages (compact), pages given back (free).
//
// refs[p] counts the table entries that name page p; 0 is a free page. A row of a table names its sequence's pages from block 0 on
// and -1 behind them. The book-keeping kernels are bound by the chain of their dependent loads (0.6 to 0.8 us each), the copies by HBM.
#include "memory.cuh"
#include "tc.cuh"

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
// Row b becomes what row parent[b] was, all rows at once. A CTA takes C of the table's columns, all rows of them staged in shared memory, so
// that rows may change places in the table itself. Every CTA reads the lengths; they are changed when all have: behind the barrier of
// a cluster where eight CTAs hold the table (`alone`), else by a second launch.
constexpr int kForkCtas = 8, kForkThreads = 512, kForkTile = 64 * 1024;

__global__ void __launch_bounds__(kForkThreads, 1) k_kv8_fork(int* __restrict__ refs, int pages, int* __restrict__ table, int blocks,
                                                              int* __restrict__ lens, const int* __restrict__ parent, int B, int shift, int alone) {
    extern __shared__ int s_mem[];
    int *s_from = s_mem, *s_len = s_mem + B, *s_tile = s_mem + 2 * B;      // parent, tokens of the row's old sequence, a tile
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, C = 1 << shift, c0 = blockIdx.x * C;
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
    if (alone) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const int n = c0 < blocks ? B << shift : 0;
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
    if (!alone) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (blockIdx.x == 0)
        for (int b = tid; b < B; b += kForkThreads) lens[b] = s_from[b] < 0 ? 0 : s_len[s_from[b]];
}

// The lengths after a fork whose table more CTAs have changed.
__global__ void __launch_bounds__(kForkThreads, 1) k_kv8_fork_lens(int* __restrict__ lens, const int* __restrict__ parent, int B, int most) {
    extern __shared__ int s_mem[];
    pdl_launch_dependents();
    pdl_wait();
    for (int b = threadIdx.x; b < B; b += kForkThreads) s_mem[b] = min(max(lens[b], 0), most);
    __syncthreads();
    for (int b = threadIdx.x; b < B; b += kForkThreads) {
        const int p = parent[b] >= B ? b : parent[b];
        lens[b] = p < 0 ? 0 : s_mem[p];
    }
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

// Where a page's writers are counted: open addressing in shared memory, at least two places to a sequence.
struct Writers {
    int *page, *count, *last;
    u32 mask;
    TCQ_HD u32 place(int p) const {
        u32 i = ((u32)p * 2654435761u >> 7) & mask;
        for (;;) {
            const int seen = atomicCAS(page + i, -1, p);
            if (seen == -1 || seen == p) return i;
            i = (i + 1) & mask;
        }
    }
};

__global__ void __launch_bounds__(kResThreads, 1) k_kv8_reserve(int* refs, int pages, int* __restrict__ table, int blocks,
                                                                const int* __restrict__ lens, const int* __restrict__ count,
                                                                int* __restrict__ granted, int* __restrict__ copies, int B, int lanes, int places) {
    extern __shared__ int s_mem[];
    // missing pages up to a sequence, its first missing block, its begun block's page
    int *s_upto = s_mem, *s_first = s_mem + B, *s_begun = s_mem + 2 * B;
    const Writers W = {s_mem + 3 * B, s_mem + 3 * B + places, s_mem + 3 * B + 2 * places, (u32)places - 1};
    __shared__ int s_warp[32];
    const int tid = threadIdx.x, sub = tid & (lanes - 1), per_pass = kResThreads / lanes;
    for (int i = tid; i < places; i += kResThreads) W.page[i] = W.last[i] = -1, W.count[i] = 0;
    pdl_launch_dependents();
    pdl_wait();
    const int limit = (int)min((i64)blocks * kBlk, (i64)0x7fffffff);
    const u32 mask0 = free_mask(refs, pages, (i64)tid * kResPer);
    __syncthreads();
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
                if (begun) at = table[(i64)b * blocks + first];
                for (int j = first + begun + sub; j < last; j += lanes) missing += table[(i64)b * blocks + j] < 0;
                if (begun && (unsigned)at >= (unsigned)pages) fits = false, at = -1;
            }
        }
        for (int o = 1; o < lanes; o <<= 1) missing += __shfl_xor_sync(0xffffffffu, missing, o);
        if (b < B && sub == 0) {
            if (!fits) out_of_range();
            const bool want = cnt > 0 && fits;
            s_upto[b] = want ? missing : -1;                                // -1: nothing asked for, or no room in the table
            s_first[b] = want ? last - missing : 0;
            if (want && at >= 0) {
                const u32 w = W.place(at);
                atomicAdd(W.count + w, 1);
                atomicMax(W.last + w, b);
            }
            s_begun[b] = want ? at : -1;
        }
    }
    __syncthreads();
    // A page that others name too is replaced for its writers; where the writers are all who name it, the last of them keeps it.
    for (int b = tid; b < B; b += kResThreads) {
        const int at = s_begun[b];
        if (at < 0) continue;
        const int held = __ldcg(refs + at);
        const u32 w = W.place(at);
        if (held <= 1 || (held == W.count[w] && W.last[w] == b)) s_begun[b] = -1;
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
        if (ok && copied) atomicAdd(refs + s_begun[b], -1);
        refused |= asked && !ok;
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

// A CTA moves 32 KB of one page's keys (blockIdx.z even) or values, eight 16-byte loads of a thread under way (256 pages of 32 KB + 32 KB in four
// layers: 14 us).
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
// A CTA writes one block of new pages, keys (blockIdx.z even) or values, in one layer, hg heads one after the other (so that the chain
// number -> page -> scale is walked once for them): for its up to 64 tokens the page and slot they come from, per head s = the
// largest of their pages' scales, q' = rint(q (s_old / s)) (a token whose page has that scale keeps its integers). Keys are rows of a
// token: a thread moves 16 bytes. Values lie token by token along a row: a thread makes words of four tokens, of one or two
// words where its warp's tokens lie four in a row (whole runs kept), else byte by byte.
//
// Quotients of integers q' = q r with 0 <= r <= 1: the byte in a float's low bits (2^23 + 128 + q), its offset taken off, times r,
// rounded to nearest even by adding 1.5 * 2^23; each step one rounding.
//
// Bound by HBM: three quarters of 2 x 65531 tokens, 8 heads of 128, four layers: 240 us of the 614 with the read back, 6.6 TB/s of what
// is kept and written; half of 4 x 16411, eight layers, 8 heads of 64: 100 us (whole rows of values are read for the half of
// them). With source tiles in shared memory and a CTA for each head about 350 and 170 us.
// (The product stands alone: a packed one was contracted with the addition behind it, which rounds once and now and then to the other side.)
TCQ_HD u32 scaled4(u32 w, const float4& r) {
    const u32 u = w ^ 0x80808080u, c = 0x4b000000u;
    const u64 off = pair(-8388736.f, -8388736.f), big = pair(12582912.f, 12582912.f);
    const u64 a = pair(__uint_as_float(__byte_perm(u, c, 0x7440)), __uint_as_float(__byte_perm(u, c, 0x7441)));
    const u64 b = pair(__uint_as_float(__byte_perm(u, c, 0x7442)), __uint_as_float(__byte_perm(u, c, 0x7443)));
    float x, y, z, v;
    unpair(add2(a, off), x, y);
    unpair(add2(b, off), z, v);
    unpair(add2(pair(__fmul_rn(x, r.x), __fmul_rn(y, r.y)), big), x, y);
    unpair(add2(pair(__fmul_rn(z, r.z), __fmul_rn(v, r.w)), big), z, v);
    return __byte_perm(__byte_perm(__float_as_uint(x), __float_as_uint(y), 0x0040), __byte_perm(__float_as_uint(z), __float_as_uint(v), 0x0040), 0x5410);
}

constexpr int kCompactHeads = 8;

template <int D>
__global__ void __launch_bounds__(128) k_kv8_compact(const __grid_constant__ Layers L, const int* __restrict__ table, int blocks,
                                                     const int* __restrict__ lens, const int* __restrict__ index, int M,
                                                     const int* __restrict__ kept, const int* __restrict__ new_table, int new_blocks,
                                                     int pages, int heads, int NB, int hg, FastDiv by_groups, FastDiv by_blocks) {
    constexpr int TH = 128, PAGE = kBlk * D;
    __shared__ int s_page[kBlk], s_slot[kBlk];
    __shared__ __align__(16) float s_ratio[kCompactHeads][kBlk];
    __shared__ float s_top[kCompactHeads][2];
    pdl_launch_dependents();
    pdl_wait();
    const int bn = (int)fdiv(blockIdx.x, by_groups), hq = (int)blockIdx.x - bn * (int)by_groups.d, b = (int)fdiv((unsigned)bn, by_blocks),
              n = bn - b * NB, tid = threadIdx.x;
    const int h0 = hq * hg, hn = min(hg, heads - h0);
    const bool is_v = blockIdx.z & 1;
    const auto& l = L.at[blockIdx.y];
    const int slot0 = tid & (kBlk - 1), first = n * kBlk;
    // the block's tokens: numbers, pages
    int number = first + slot0 < M ? index[(i64)b * M + first + slot0] : -1;
    const int to = n < new_blocks ? new_table[(i64)b * new_blocks + n] : -1;
    int m = M;
    if (kept) {
        m = kept[b];
        if (m < 0 || m > M) {
            if (tid == 0) out_of_range();
            m = m < 0 ? 0 : M;
        }
    }
    const int len = min(lens[b], (int)min((i64)blocks * kBlk, (i64)0x7fffffff));
    const int live = min(m - first, kBlk);
    if (live <= 0) return;
    if ((unsigned)to >= (unsigned)pages) {
        if (tid == 0) out_of_range();
        return;
    }
    int page = -1;
    if (slot0 < live) {
        if (number >= 0 && number < len) page = table[(i64)b * blocks + number / kBlk];
        if ((unsigned)page >= (unsigned)pages) page = -1, out_of_range();
    }
    // scales of the heads: the first 64 threads take those of even number, the others those of odd
    const float* scale = is_v ? l.vs : l.ks;
    float sc[kCompactHeads / 2];
#pragma unroll
    for (int i = 0; i < kCompactHeads / 2; ++i) {
        const int hh = 2 * i + (tid >> 6);
        sc[i] = page >= 0 && hh < hn ? scale[(i64)page * heads + h0 + hh] : 0.f;
    }
    if (tid < kBlk) s_page[tid] = page, s_slot[tid] = number & (kBlk - 1);
#pragma unroll
    for (int i = 0; i < kCompactHeads / 2; ++i) {
        float top = sc[i];
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((tid & 31) == 0) s_top[2 * i + (tid >> 6)][tid >> 5 & 1] = top;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kCompactHeads / 2; ++i) {
        const int hh = 2 * i + (tid >> 6);
        const float top = fmaxf(s_top[hh][0], s_top[hh][1]);
        s_ratio[hh][slot0] = top > 0.f ? sc[i] / top : 0.f;
        if (slot0 == 0 && hh < hn) (is_v ? l.vs : l.ks)[(i64)to * heads + h0 + hh] = top;
    }
    const i64 dst = ((i64)to * heads + h0) * PAGE;
    __syncthreads();
    if (!is_v) {
        constexpr int C = D / 16, NU = (kBlk * C + TH - 1) / TH;
        const i8* src[NU];
        bool there[NU];
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = tid + TH * i, t = min(u / C, kBlk - 1), c = u - u / C * C, p = s_page[t];
            there[i] = p >= 0 && u < kBlk * C;
            src[i] = l.k + ((i64)max(p, 0) * heads + h0) * PAGE + s_slot[t] * D + 16 * c;
        }
#pragma unroll 2
        for (int hh = 0; hh < hn; ++hh) {
            uint4 w[NU];
#pragma unroll
            for (int i = 0; i < NU; ++i) w[i] = there[i] ? *reinterpret_cast<const uint4*>(src[i] + hh * PAGE) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int u = tid + TH * i, t = u / C;
                if (kBlk * C % TH != 0 && u >= kBlk * C) break;
                const float r = s_ratio[hh][t];
                if (r != 1.f) {
                    const float4 r4 = make_float4(r, r, r, r);
                    w[i].x = scaled4(w[i].x, r4), w[i].y = scaled4(w[i].y, r4), w[i].z = scaled4(w[i].z, r4), w[i].w = scaled4(w[i].w, r4);
                }
                *reinterpret_cast<uint4*>(l.k + dst + hh * PAGE + 16 * u) = w[i];
            }
        }
        return;
    }
    // Values: word (d, g) holds tokens 4 g .. 4 g + 3 of element d; sixteen lanes to a row.
    constexpr int NW = D * 16 / TH, ROWS = TH / 16;
    const int g = tid & 15, d0 = tid >> 4;
    const i8* src[4];
    bool there[4], run = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int p = s_page[4 * g + e], s = s_slot[4 * g + e];
        there[e] = p >= 0;
        src[e] = l.v + ((i64)max(p, 0) * heads + h0) * PAGE + d0 * kBlk + s;
        run = run && src[e] == src[0] + e && there[e] == there[0];
    }
    run = run || !(there[0] || there[1] || there[2] || there[3]);
    const u32 skew = (u32)(reinterpret_cast<uintptr_t>(src[0]) & 3);
    const u32* word = reinterpret_cast<const u32*>(src[0] - skew);
    const bool words = __all_sync(0xffffffffu, run);
#pragma unroll 1
    for (int hh = 0; hh < hn; ++hh) {
        u32 out[NW];
        if (words) {
            u32 more[NW];
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                out[i] = there[0] ? word[hh * (PAGE / 4) + ROWS * i * (kBlk / 4)] : 0u;
                more[i] = there[0] && skew ? word[hh * (PAGE / 4) + ROWS * i * (kBlk / 4) + 1] : 0u;
            }
#pragma unroll
            for (int i = 0; i < NW; ++i) out[i] = __funnelshift_r(out[i], more[i], 8 * skew);
        } else {
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                u32 x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = there[e] ? (unsigned char)src[e][hh * PAGE + ROWS * i * kBlk] : 0u;
                out[i] = __byte_perm(x[0] | x[1] << 8, x[2] | x[3] << 8, 0x5410);
            }
        }
        const float4 r = *reinterpret_cast<const float4*>(&s_ratio[hh][4 * g]);
        if (r.x != 1.f || r.y != 1.f || r.z != 1.f || r.w != 1.f) {
#pragma unroll
            for (int i = 0; i < NW; ++i) out[i] = scaled4(out[i], r);
        }
        u32* const to_v = reinterpret_cast<u32*>(l.v + dst + hh * PAGE) + d0 * 16 + g;
#pragma unroll
        for (int i = 0; i < NW; ++i) to_v[ROWS * 16 * i] = out[i];
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
    // columns of a CTA: eight (a sector of the table), four where eight CTAs hold the whole table then, fewer where all rows' would not fit
    int shift = blocks <= 4 * kForkCtas ? 2 : 3;
    while (shift > 0 && ((i64)B << shift) * 4 > kForkTile) --shift;
    const int ctas = (blocks + (1 << shift) - 1) >> shift, alone = ctas <= kForkCtas;
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return TCQ_ERR_DEVICE;
    constexpr int most = kForkTile + 8 * TCQ_KV8_MAX_SEQUENCES;
    if (!(set.load(std::memory_order_relaxed) >> dev & 1)) {
        if (cudaFuncSetAttribute(k_kv8_fork, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) return TCQ_ERR_LAUNCH;
        set.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kForkThreads);
    cfg.dynamicSmemBytes = (size_t)4 * (((size_t)B << shift) + 2 * B);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = alone ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, k_kv8_fork, (int*)refs, pages, (int*)table, blocks, (int*)lens, (const int*)parent, B, shift, alone) != cudaSuccess)
        return TCQ_ERR_LAUNCH;
    const i64 tokens = (i64)blocks * kBlk;
    return alone ? TCQ_OK : launch_pdl(k_kv8_fork_lens, dim3(1), kForkThreads, (size_t)4 * B, stream, (int*)lens, (const int*)parent, B,
                                       (int)(tokens < 0x7fffffff ? tokens : 0x7fffffff));
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
    int places = 64;
    while (places < 2 * B) places <<= 1;
    constexpr int most = 36 * TCQ_KV8_MAX_SEQUENCES;
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return TCQ_ERR_DEVICE;
    if (!(set.load(std::memory_order_relaxed) >> dev & 1)) {
        if (cudaFuncSetAttribute(k_kv8_reserve, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) return TCQ_ERR_LAUNCH;
        set.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return launch_pdl(k_kv8_reserve, dim3(1), kResThreads, (size_t)12 * (B + places), stream, (int*)refs, pages, (int*)table, blocks, (const int*)lens,
                      (const int*)count, (int*)granted, (int*)copies, B, lanes, places);
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
    // heads that a CTA takes one after the other: fewer where the launch would be short of CTAs
    int hg = kCompactHeads;
    while (hg > 1 && (i64)B * NB * ((heads + hg - 1) / hg) * (layers < TCQ_KV8_MAX_LAYERS ? layers : TCQ_KV8_MAX_LAYERS) * 2 < (i64)16 * tcq_sm_count()) hg >>= 1;
    const int groups = (heads + hg - 1) / hg;
    const i64 ctas = (i64)B * NB * groups;
    if (ctas > 0x7fffffff) return TCQ_ERR_SHAPE;
    const FastDiv by_groups = make_fastdiv((unsigned)groups), by_blocks = make_fastdiv((unsigned)NB);
    return by_layers(caches, layers, [&](int count, const Layers& L) {
        return by_head_dim(caches->head_dim, [&](auto d) {
            return launch_pdl(k_kv8_compact<decltype(d)::value>, dim3((unsigned)ctas, count, 2), 128, 0, stream, L, (const int*)table, blocks,
                              (const int*)lens, (const int*)index, tokens, (const int*)kept, (const int*)new_table, new_blocks,
                              caches->pages, heads, NB, hg, by_groups, by_blocks);
        });
    });
}

}  // extern "C"
