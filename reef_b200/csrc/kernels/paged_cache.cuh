// Page tables from the lengths of the requests, and the append of new keys and values to the paged cache.
// The reference serves no model that keeps state between tokens; these stand beside its BERT kernels as what a decoder needs.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "simple.cuh"

namespace reef {

__device__ __forceinline__ int page_of(const PagedP& p, int pos) { return (int)(__umulhi((unsigned)pos << 1, p.ps_mul) >> p.ps_shift); }

// ---- page tables ---------------------------------------------------------------------------------------------------------
// args: table, lens, new, [parent], table', lens', start, tok, status, [fork].
// Row r goes on from row q = parent[r] (itself without parents; -1: from nothing), holds l = lens[q] tokens and adds n = new[r].
// It keeps the first ceil(l / ps) pages of q, and gets ceil((l + n) / ps) - ceil(l / ps) free ones; one more replaces a last page
// that is partly filled and that a lower row with the same parent keeps, and `fork` says what is to be copied into it.  So no
// two rows ever share a page that one of them will write.  Free is what no row keeps; lowest ids first, rows in their order.
// A row that cannot be served is refused (status 2: lengths, parent or ids out of range; 3: more than `tokens` new tokens in all;
// 1: no pages left) and comes out empty.  Tokens are counted over the rows that are not 2, and all of them are 3 from the one on that
// goes beyond; pages over the rows left, and those that need any are 1 from the one on that goes beyond.
// The state goes from one set of buffers into another, so the kernel can be run again after a preemption.
//
// Nothing here moves many bytes: the time is that of the dependent steps (lengths, ids, prefix sums, rows).  The allocation is
// worked out by every block for itself (no block has to wait for another); each block then writes its own share of the rows.
constexpr int kTablesMaxRows = 1024, kTablesMaxPages = 1 << 19;
__host__ __device__ inline int tables_words(int pages) { return (pages + 31) / 32; }
__host__ constexpr int tables_smem(int rows, int pages) { return 4 * ((pages + 31) / 32 + 6 * rows + 2 + 32); }
constexpr int kTablesSmemMax = tables_smem(kTablesMaxRows, kTablesMaxPages);

__device__ __forceinline__ int block_scan(int v, int* sums, int* total) {   // inclusive, over 256 threads in their order
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 8; w++) {
        if (w < warp) before += sums[w];
        all += sums[w];
    }
    *total = all;
    return v + before;
}

__device__ __forceinline__ bool body_page_tables(const KTask& t, int vb, unsigned char* smem, const int*) {
    const PagedP& p = t.p.paged;
    const int R = p.rows, M = p.mp, S = p.ps, N = p.pages, f = p.has_fork;
    const int* table = (const int*)t.a[0];
    const int* lens = (const int*)t.a[1];
    const int* fresh = (const int*)t.a[2];
    const int* parent = f ? (const int*)t.a[3] : nullptr;
    int* table_out = (int*)t.a[3 + f];
    int* lens_out = (int*)t.a[4 + f];
    int* start_out = (int*)t.a[5 + f];
    int4* tok_out = (int4*)t.a[6 + f];
    int* status_out = (int*)t.a[7 + f];
    int4* fork_out = f ? (int4*)t.a[9] : nullptr;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, words = tables_words(N);
    unsigned* used = (unsigned*)smem;              // a bit per page
    int* sums = (int*)(used + words);              // 32 words of scratch
    int* len = sums + 32;                          // per row: tokens held
    int* add = len + R;                            // tokens added
    int* from = add + R;                           // row it goes on from
    int* state = from + R;                         // status; then (accepted rows) 0
    int* base = state + R;                         // rank of its first new page among the free ones [R + 1]
    int* begin = base + R + 1;                     // first token [R + 1], also the lowest child of a row on the way
    __syncthreads();                               // a persistent caller's previous block is out of shared memory
    for (int i = tid; i < words; i += kThreads) used[i] = 0;
    for (int r = tid; r < R; r += kThreads) {
        const int q = f ? parent[r] : r;
        const bool named = q >= -1 && q < R;
        const int l = named && q >= 0 ? lens[q] : 0, n = fresh[r];
        const bool good = named && l >= 0 && n >= 0 && (long long)l + n <= (long long)M * S;
        len[r] = l; add[r] = n; from[r] = q;
        state[r] = good ? 0 : 2;
        begin[r] = R;
    }
    __syncthreads();
    // ids of the rows, a row to a warp: in range, and marked as used only where the whole row is good
    for (int r = warp; r < R; r += 8) {
        if (state[r]) continue;
        const int l = len[r], kept = page_of(p, l + S - 1);
        const int* ids = table + (size_t)max(from[r], 0) * M;
        bool bad = false;
        for (int j = lane; j < kept; j += 32) {
            const int id = ids[j];
            bad |= id < -1 || id >= N || (id < 0 && j == kept - 1 && l != kept * S);
        }
        bad = __any_sync(0xffffffffu, bad);
        if (bad) {
            if (lane == 0) state[r] = 2;
            continue;
        }
        for (int j = lane; j < kept; j += 32) {
            const int id = ids[j];
            if (id >= 0) atomicOr(&used[id >> 5], 1u << (id & 31));
        }
        if (f && lane == 0 && from[r] >= 0) atomicMin(&begin[from[r]], r);
    }
    __syncthreads();
    // sums over the rows: tokens, then pages of those whose tokens have room
    const int per = (R + kThreads - 1) / kThreads, r0 = tid * per, r1 = min(R, r0 + per);
    int part = 0, all, have = 0;
    const int wper = (words + kThreads - 1) / kThreads, w0 = tid * wper, w1 = min(words, w0 + wper);
    for (int w = w0; w < w1; w++) have += __popc(used[w]);
    const int holes = max(0, min(N, w1 * 32) - w0 * 32) - have;     // free pages among this thread's words
    int frees;
    const int hole0 = block_scan(w0 < w1 ? holes : 0, sums, &frees) - (w0 < w1 ? holes : 0);
    // (a length is at most 2^30, a sum over the rows goes beyond 32 bits: it stops counting where it is beyond any room)
    auto clipped = [](int a, int b) { return (int)min((long long)a + b, 0x1fffffLL); };
    for (int r = r0; r < r1; r++) part = clipped(part, state[r] == 0 ? add[r] : 0);
    int upto = block_scan(part, sums, &all) - part;
    for (int r = r0; r < r1; r++) {
        if (state[r]) continue;
        upto = clipped(upto, add[r]);
        if (upto > p.tokens) state[r] = 3;
    }
    auto forked = [&](int r) { return f && state[r] == 0 && from[r] >= 0 && len[r] != page_of(p, len[r]) * S && begin[from[r]] != r; };
    auto needs = [&](int r) { return state[r] ? 0 : page_of(p, len[r] + add[r] + S - 1) - page_of(p, len[r] + S - 1) + (forked(r) ? 1 : 0); };
    part = 0;
    for (int r = r0; r < r1; r++) part = clipped(part, needs(r));
    upto = block_scan(part, sums, &all) - part;
    const int want = min(all, frees);
    for (int r = r0; r < r1; r++) {
        const int n = needs(r);
        base[r] = upto;
        upto = clipped(upto, n);
        if (n > 0 && upto > frees) state[r] = 1;
    }
    if (tid == 0) base[R] = all;
    part = 0;
    for (int r = r0; r < r1; r++) part += state[r] ? 0 : add[r];
    upto = block_scan(part, sums, &all) - part;
    // this block's rows; the lowest children are read for the last time
    const int rows_per = (R + p.split - 1) / p.split, mine0 = min(R, vb * rows_per), mine1 = min(R, mine0 + rows_per);
    unsigned fork_bits = 0;                         // of this thread's rows (at most four)
    for (int r = r0; r < r1; r++) fork_bits |= forked(r) ? 1u << (r - r0) : 0;
    __syncthreads();
    for (int r = r0; r < r1; r++) {
        begin[r] = upto;
        upto += state[r] ? 0 : add[r];
        if (state[r]) len[r] = add[r] = 0, from[r] = -1;
        if (fork_bits >> (r - r0) & 1) state[r] = -1;   // accepted, with a copy
    }
    if (tid == kThreads - 1) begin[R] = all;
    __syncthreads();
    // kept pages and the empty rest, a row to a warp
    for (int r = mine0 + warp; r < mine1; r += 8) {
        const int q = from[r], kept = page_of(p, len[r] + S - 1), total = page_of(p, len[r] + add[r] + S - 1);
        const int copied = state[r] < 0 ? kept - 1 : kept;
        const int* ids = table + (size_t)max(q, 0) * M;
        for (int j = lane; j < M; j += 32)
            if (j < copied || j >= total) table_out[(size_t)r * M + j] = j < copied ? ids[j] : -1;
    }
    // free pages by rank: every thread's words hold the ranks from hole0 on
    if (hole0 < want) {
        int rank = hole0, r = 0;
        {   // the last row that begins at or before this rank
            int hi = R;
            while (hi - r > 1) {
                const int mid = (r + hi) >> 1;
                if (base[mid] <= rank) r = mid; else hi = mid;
            }
        }
        for (int w = w0; w < w1 && rank < want; w++) {
            unsigned open = ~used[w];
            if (w == words - 1 && (N & 31)) open &= (1u << (N & 31)) - 1;
            while (open && rank < want) {
                const int id = w * 32 + __ffs(open) - 1;
                open &= open - 1;
                while (r + 1 < R && base[r + 1] <= rank) r++;
                if (r >= mine0 && r < mine1 && state[r] <= 0) {
                    const int j = page_of(p, len[r] + S - 1) + (state[r] < 0 ? -1 : 0) + rank - base[r];
                    if (j < M) table_out[(size_t)r * M + j] = id;
                }
                rank++;
            }
        }
    }
    __syncthreads();
    for (int r = mine0 + tid; r < mine1; r += kThreads) {
        lens_out[r] = len[r] + add[r];
        start_out[r] = begin[r];
        status_out[r] = max(state[r], 0);
        if (f) {
            const int kept = page_of(p, len[r] + S - 1);
            int4 c = make_int4(-1, -1, 0, 0);
            if (state[r] < 0) c = make_int4(table[(size_t)from[r] * M + kept - 1], table_out[(size_t)r * M + kept - 1], len[r] - (kept - 1) * S, 0);
            fork_out[r] = c;
        }
    }
    if (vb == 0 && tid == 0) start_out[R] = begin[R];
    for (int i = begin[mine0] + tid; i < begin[mine1]; i += kThreads) {
        int r = mine0, hi = mine1;
        while (hi - r > 1) {
            const int mid = (r + hi) >> 1;
            if (begin[mid] <= i) r = mid; else hi = mid;
        }
        const int pos = len[r] + i - begin[r], j = page_of(p, pos);
        tok_out[i] = make_int4(table_out[(size_t)r * M + j] * S + pos - j * S, r, pos + 1, 0);
    }
    for (int i = begin[R] + vb * kThreads + tid; i < p.tokens; i += p.split * kThreads) tok_out[i] = make_int4(-1, -1, 0, 0);
    return true;
}

// ---- append --------------------------------------------------------------------------------------------------------------
// args: k, v, tok, [fork], k_cache, v_cache.  cache[slot / ps][head][slot % ps][:] = k[token][head][:], rounded to the cache's type
// (to nearest even: the type is the caller's choice); tokens without a slot are passed over.  A fork (src, dst, n) copies the
// first n tokens of a page; new tokens are written behind them, and src's first n are written by nobody, so the order of the
// two does not matter and a second run gives the same.  Bound by HBM: every byte is moved once, 16 at a time.
constexpr int kAppendPerBlock = 4 * kThreads * 4;       // fp32 values of k, and of v
__host__ inline int append_token_blocks(const PagedP& p) {
    return (int)(((long long)p.tokens * p.kvh * p.d + kAppendPerBlock - 1) / kAppendPerBlock);
}
__host__ inline int append_fork_blocks(const PagedP& p) { return p.has_fork ? (p.rows * p.kvh + 3) / 4 : 0; }

__device__ __forceinline__ void store4(float* at, float4 x) { *reinterpret_cast<float4*>(at) = x; }
__device__ __forceinline__ void store4(__nv_bfloat16* at, float4 x) {
    union { __nv_bfloat162 h[2]; uint2 u; } y;
    y.h[0] = __floats2bfloat162_rn(x.x, x.y);
    y.h[1] = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(at) = y.u;
}
__device__ __forceinline__ void store4(__half* at, float4 x) {
    union { __half2 h[2]; uint2 u; } y;
    y.h[0] = __floats2half2_rn(x.x, x.y);
    y.h[1] = __floats2half2_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(at) = y.u;
}

template <class C>
__device__ __forceinline__ void append_tokens(const PagedP& p, const KTask& t, int vb) {
    const float* k = (const float*)t.a[0] + p.qo;
    const float* v = (const float*)t.a[1] + p.vo;
    const int4* tok = (const int4*)t.a[2];
    C* kc = (C*)t.a[3 + p.has_fork];
    C* vc = (C*)t.a[4 + p.has_fork];
    const int row = p.kvh * p.d, row4 = row >> 2;
    const long long total = (long long)p.tokens * row4;
    float4 a[4], b[4];
    C *ka[4], *va[4];
#pragma unroll
    for (int it = 0; it < 4; it++) {
        const long long i = (long long)vb * (kAppendPerBlock / 4) + it * kThreads + threadIdx.x;
        ka[it] = nullptr;
        if (i >= total) continue;
        const int token = (int)(i / row4), c = (int)(i - (long long)token * row4) << 2, h = c / p.d, e = c - h * p.d;
        const int slot = tok[token].x;
        if (slot < 0 || slot >= p.pages * p.ps) continue;
        const int page = page_of(p, slot);
        const size_t at = (((size_t)page * p.kvh + h) * p.ps + (slot - page * p.ps)) * p.d + e;
        ka[it] = kc + at;
        va[it] = vc + at;
        a[it] = *reinterpret_cast<const float4*>(k + (size_t)token * p.qs + c);
        b[it] = *reinterpret_cast<const float4*>(v + (size_t)token * p.vs + c);
    }
#pragma unroll
    for (int it = 0; it < 4; it++)
        if (ka[it]) {
            store4(ka[it], a[it]);
            store4(va[it], b[it]);
        }
}

__device__ __forceinline__ bool body_paged_append(const KTask& t, int vb, unsigned char*, const int*) {
    const PagedP& p = t.p.paged;
    if (vb < p.split) {
        if (p.kt == KT_FP32) append_tokens<float>(p, t, vb);
        else if (p.kt == KT_BF16) append_tokens<__nv_bfloat16>(p, t, vb);
        else append_tokens<__half>(p, t, vb);
        return true;
    }
    // forks: two warps to a head of a forked page, one for keys and one for values
    const int4* fork = (const int4*)t.a[3];
    const int item = (vb - p.split) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 31;
    if (item >= p.rows * p.kvh) return true;
    const int r = item / p.kvh, h = item - r * p.kvh;
    const int4 c = fork[r];
    if ((unsigned)c.x >= (unsigned)p.pages || (unsigned)c.y >= (unsigned)p.pages || c.x == c.y) return true;
    const int e = p.kt == KT_FP32 ? 4 : 2, words = min(c.z, p.ps) * (p.d * e / 16);
    const size_t page = (size_t)p.ps * p.d * e;
    char* cache = (char*)t.a[threadIdx.x & 32 ? 5 : 4];
    const uint4* src = (const uint4*)(cache + ((size_t)c.x * p.kvh + h) * page);
    uint4* dst = (uint4*)(cache + ((size_t)c.y * p.kvh + h) * page);
#pragma unroll 4
    for (int i = lane; i < words; i += 32) dst[i] = src[i];
    return true;
}

}  // namespace reef
