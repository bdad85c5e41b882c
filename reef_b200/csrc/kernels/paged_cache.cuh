// Page tables from the lengths of the requests, and the append of new keys and values to the paged cache.
// The reference serves no model that keeps state between tokens; these stand beside its BERT kernels as what a decoder needs.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "simple.cuh"

namespace reef {

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two fp32 values at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 z, x, y, z;\n\t"
        "mov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ int page_of(const PagedP& p, int pos) { return (int)(__umulhi((unsigned)pos << 1, p.ps_mul) >> p.ps_shift); }

// ---- page tables ---------------------------------------------------------------------------------------------------------
// args: table, lens, new, [parent], table', lens', start, tok, status, [fork].
// Row r goes on from row q = parent[r] (itself without parents; -1: from nothing), holds l = lens[q] tokens and adds n = new[r].
// It keeps the first ceil(l / ps) pages of q, and gets ceil((l + n) / ps) - ceil(l / ps) free ones; one more replaces a last page
// that is partly filled and that a lower row with the same parent keeps, and `fork` says what is to be copied into it.  So no
// two rows ever share a page that one of them will write.  Free is what no row keeps; lowest ids first, rows in their order.
// A row that cannot be served is refused (status 2: lengths, parent or ids out of range; 3: more than `tokens` new tokens in all;
// 1: no pages left) and comes out empty.  With 1 and 3 what it kept stays in use in this step, with 2 it keeps nothing.  Tokens are counted over the rows that are not 2, and all of them are 3 from the one on that
// goes beyond; pages over the rows left, and those that need any are 1 from the one on that goes beyond.
// The state goes from one set of buffers into another, so the kernel can be run again after a preemption.
//
// Nothing here moves many bytes: the time is that of the dependent steps (lengths, ids, prefix sums, ids again).  The allocation is
// worked out by every block for itself, so that no block has to wait for another; the rows and tokens to write are divided.  Ids are read in
// pieces of 128 of a row, eight pieces of a warp under way whatever the rows' lengths, and parents that several rows go on from once.
// Used pages are marked in bytes, a window of the pages at a time, and packed to bits: an atomic OR into a word of bits took 1.5 cycles for
// every id, 53 us for 62500 of them, a byte is a plain store.  A free page is found by its rank (a prefix sum over the threads' words, a walk
// through one thread's), by whoever needs it.  16 rows of 500 tokens 7 us, 128 beams 12, 256 rows of two million tokens in all (62500 ids)
// 21 (86 with atomics, rows one after the other, and free pages handed out by the threads whose words hold them), 1024 rows of 524288 in all
// in a pool of as many, which takes five windows and the ids five times, 444.
constexpr int kTablesThreads = 2 * kThreads;
constexpr int kTablesMaxRows = 1024, kTablesMaxPages = 1 << 19;
__host__ __device__ constexpr int tables_fixed(int rows, int pages) {
    return (4 * ((pages + 31) / 32 + 8 * rows + 2 + 96 + kTablesThreads) + 15) / 16 * 16;
}
__host__ __device__ constexpr int tables_window(int rows, int pages) {      // what fits an SM beside the rest
    const int all = (pages + 31) / 32 * 32, room = (225 * 1024 - tables_fixed(rows, pages)) / 512 * 512;
    return all < room ? all : room;
}
__host__ constexpr int tables_smem(int rows, int pages) { return tables_fixed(rows, pages) + tables_window(rows, pages); }
constexpr int kTablesSmemMax = 225 * 1024;
// Twice the threads from 8192 ids on: 64 rows of 512 ids 12.4 us instead of 14.4, 256 rows of 1024 20.6 instead of 26.8, 16 rows of 64
// 10.4 instead of 9.0.  With 1024 threads barriers and sums cost more than is divided: 16.5, 24.3 and 12.4.  A dispatcher's
// blocks, which have kThreads, do the same work.
__host__ inline int tables_threads(int rows, int max_pages) { return (long long)rows * max_pages >= 8192 ? kTablesThreads : kThreads; }
// Rows and tokens are written by up to 32 blocks, 4096 ids or 256 tokens to a block.
__host__ inline int tables_blocks(int rows, int max_pages, int tokens) {
    const long long want = max(((long long)rows * max_pages + 4095) / 4096, (long long)(tokens + 255) / 256);
    return (int)min(want, 32LL);
}

// sums over a block's threads in their order, of N values side by side; returns the exclusive ones in v, the totals in all
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&all)[N], int* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int x[N], y[N];
    auto scan = [&](int (&z)[N]) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int u = __shfl_up_sync(0xffffffffu, z[n], o);
                if (lane >= o) z[n] += u;
            }
        }
    };
#pragma unroll
    for (int n = 0; n < N; n++) x[n] = v[n];
    scan(x);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; n++)
        if (lane == 31) sums[32 * n + warp] = x[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; n++) y[n] = lane < warps ? sums[32 * n + lane] : 0;
    scan(y);
#pragma unroll
    for (int n = 0; n < N; n++) {
        const int before = __shfl_sync(0xffffffffu, y[n], max(warp - 1, 0));
        all[n] = __shfl_sync(0xffffffffu, y[n], 31);
        v[n] = x[n] - v[n] + (warp ? before : 0);
    }
}
// the last i in [lo, hi) with a[i] <= x (a does not fall, a[lo] <= x)
__device__ __forceinline__ int last_below(const int* a, int lo, int hi, int x) {
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
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
    const int threads = blockDim.x, warps = threads >> 5, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, words = (N + 31) / 32;
    unsigned* open = (unsigned*)smem;              // a bit per page: used, later free
    int* sums = (int*)(open + words);              // scratch of the prefix sums
    int* holes = sums + 96;                        // free pages before every thread's words
    int* len = holes + kTablesThreads;                      // per row: tokens held
    int* add = len + R;                            // tokens added
    int* from = add + R;                           // row it goes on from, -1 for none
    int* state = from + R;                         // status; -1 accepted with a copy of the last page
    int* owner = state + R;                        // per parent: the lowest row that goes on from it
    int* bad = owner + R;                          // per parent: an id out of range
    int* base = bad + R;                           // rank of a row's first new page among the free ones [R + 1]; pieces of 32 ids before
    int* begin = base + R + 1;                     // its first token [R + 1]
    unsigned char* mark = smem + tables_fixed(R, N);      // a byte per page of a window
    const int window = tables_window(R, N);
    const bool wide = (M & 3) == 0 && ((uintptr_t)table & 15) == 0;         // rows begin at 16-byte boundaries
    __syncthreads();                               // a persistent caller's previous block is out of shared memory
    for (int r = tid; r < R; r += threads) {
        const int q = f ? parent[r] : r;
        const bool named = q >= -1 && q < R;
        const int l = named && q >= 0 ? lens[q] : 0, n = fresh[r];
        const bool good = named && l >= 0 && n >= 0 && (long long)l + n <= (long long)M * S;
        len[r] = l; add[r] = n; from[r] = good ? q : -1;
        state[r] = good ? 0 : 2;
        owner[r] = f ? R : r;
        bad[r] = 0;
    }
    __syncthreads();
    if (f) {
        for (int r = tid; r < R; r += threads)
            if (from[r] >= 0) atomicMin(&owner[from[r]], r);
        __syncthreads();
    }
    // a thread's rows in their order
    const int per = (R + threads - 1) / threads, r0 = tid * per, r1 = min(R, r0 + per);
    auto kept = [&](int r) { return page_of(p, len[r] + S - 1); };
    auto pieces = [&](int r) { return state[r] == 0 && from[r] >= 0 && owner[from[r]] == r ? (kept(r) + 127) >> 7 : 0; };
    // bits of the pages that no row keeps; `part` of them among this thread's words
    const int wper = (words + threads - 1) / threads, w0 = min(words, tid * wper), w1 = min(words, w0 + wper);
    int part[3] = {0, 0, 0}, all[3];
    for (int pass = 0; pass < 2; pass++) {         // (a second time without the rows whose ids are out of range, if there are any)
        int count1[1] = {0}, all1[1];
        for (int r = r0; r < r1; r++) count1[0] += pieces(r);
        block_scan(count1, all1, sums);
        for (int r = r0; r < r1; r++) {
            base[r] = count1[0];
            count1[0] += pieces(r);
        }
        if (tid == 0) base[R] = all1[0];
        bool wrong = false;
        for (int first = 0; first < N; first += window) {
            for (int i = tid * 16; i < window; i += threads * 16) *reinterpret_cast<uint4*>(mark + i) = make_uint4(0, 0, 0, 0);
            __syncthreads();
            for (int c0 = 0; c0 < all1[0]; c0 += threads) {
                // the pieces go round the warps, 32 of them at a time: a lane looks up the row of one
                const int c = c0 + warp + warps * lane;
                int at = 0, left = 0, row = 0;
                if (c < all1[0]) {
                    row = last_below(base, 0, R, c);
                    const int j = (c - base[row]) * 128;
                    left = min(kept(row) - j, 129);
                    at = from[row] * M + j;                                             // (rows * max_pages is at most 2^30)
                    if (left <= 128 && len[row] != kept(row) * S) left |= 1 << 30;     // its last id names a page that is written
                }
                const int n = min(32, (all1[0] - c0 - warp + warps - 1) / warps);
                auto look = [&](auto at_once, int i0) {
                    constexpr int P = decltype(at_once)::value;
                    int4 id[P];
                    int count[P];
                    unsigned ill = 0;
#pragma unroll
                    for (int i = 0; i < P; i++) {
                        const int* from4 = table + __shfl_sync(0xffffffffu, at, i0 + i) + 4 * lane;
                        count[i] = __shfl_sync(0xffffffffu, left, i0 + i);       // (0 behind the last piece)
                        const int m = min(count[i] & ~(1 << 30), 128) - 4 * lane;
                        id[i] = make_int4(-1, -1, -1, -1);
                        if (wide) {
                            // (what lies behind the row's last id is looked away from below; the row of the table ends at 16 bytes)
                            if (m > 0) id[i] = *reinterpret_cast<const int4*>(from4);
                        } else {
                            if (m > 0) id[i].x = from4[0];
                            if (m > 1) id[i].y = from4[1];
                            if (m > 2) id[i].z = from4[2];
                            if (m > 3) id[i].w = from4[3];
                        }
                    }
#pragma unroll
                    for (int i = 0; i < P; i++) {
                        const int m = min(count[i] & ~(1 << 30), 128) - 4 * lane;
                        int4 x = id[i];
                        if (m > 0 && m <= 4) {                        // the row's last ids, or the piece's
                            const int end = m == 1 ? x.x : m == 2 ? x.y : m == 3 ? x.z : x.w;
                            if (count[i] >> 30 && end < 0) ill |= 1u << i;
                            if (m < 2) x.y = -1;
                            if (m < 3) x.z = -1;
                            if (m < 4) x.w = -1;
                        }
                        if (max(max(x.x, x.y), max(x.z, x.w)) >= N || min(min(x.x, x.y), min(x.z, x.w)) < -1) ill |= 1u << i;
                        const unsigned at[4] = {(unsigned)x.x - first, (unsigned)x.y - first, (unsigned)x.z - first, (unsigned)x.w - first};
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (at[e] < (unsigned)window) mark[at[e]] = 1;
                    }
                    if (__any_sync(0xffffffffu, ill)) {
                        wrong = true;
#pragma unroll 1
                        for (int i = 0; i < P; i++) {
                            const int r = __shfl_sync(0xffffffffu, row, i0 + i);
                            if (__any_sync(0xffffffffu, ill >> i & 1) && lane == 0) bad[from[r]] = 1;
                        }
                    }
                };
                if (n <= 2) look(std::integral_constant<int, 2>(), 0);        // (little code: it is fetched for one use)
                else
#pragma unroll 1
                    for (int i0 = 0; i0 < n; i0 += 8) look(std::integral_constant<int, 8>(), i0);
            }
            __syncthreads();
            for (int w = tid; w < window / 32 && first / 32 + w < words; w += threads) {
                const uint4* b = reinterpret_cast<const uint4*>(mark + w * 32);
                unsigned x = 0;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint4 y = b[h];
                    // the lowest bits of four bytes, by a product, as four bits
                    x |= ((y.x * 0x10204080u) >> 28 | (y.y * 0x10204080u) >> 28 << 4 | (y.z * 0x10204080u) >> 28 << 8 | (y.w * 0x10204080u) >> 28 << 12) << 16 * h;
                }
                x = ~x;
                if (first / 32 + w == words - 1 && (N & 31)) x &= (1u << (N & 31)) - 1;
                open[first / 32 + w] = x;
            }
            if (first + window < N) __syncthreads();       // every mark is packed before the next window clears them
        }
        if (!__syncthreads_or(wrong)) break;
        for (int r = tid; r < R; r += threads)
            if (from[r] >= 0 && bad[from[r]]) state[r] = 2;
        __syncthreads();
    }
    for (int w = w0; w < w1; w++) part[0] += __popc(open[w]);
    // sums over the rows: tokens, then pages of those whose tokens have room
    // (a length is at most 2^30, a sum over the rows goes beyond 32 bits: it stops counting where it is beyond any room)
    auto clipped = [](int a, int b) { return (int)min((long long)a + b, 0x1fffffLL); };
    auto forked = [&](int r) { return f && state[r] == 0 && from[r] >= 0 && len[r] != page_of(p, len[r]) * S && owner[from[r]] != r; };
    auto needs = [&](int r) { return state[r] ? 0 : page_of(p, len[r] + add[r] + S - 1) - kept(r) + (forked(r) ? 1 : 0); };
    auto count_rows = [&]() {
        part[1] = part[2] = 0;
        for (int r = r0; r < r1; r++) {
            part[1] = clipped(part[1], state[r] == 0 ? add[r] : 0);
            part[2] = clipped(part[2], needs(r));
        }
    };
    count_rows();
    int mine = part[0];
    block_scan(part, all, sums);
    holes[tid] = part[0];
    const int frees = all[0];
    if (all[1] > p.tokens) {
        int upto = part[1];
        for (int r = r0; r < r1; r++) {
            if (state[r]) continue;
            upto = clipped(upto, add[r]);
            if (upto > p.tokens) state[r] = 3;
        }
        count_rows();
        part[0] = mine;
        block_scan(part, all, sums);
    }
    int upto = part[2];
    for (int r = r0; r < r1; r++) {
        const int n = needs(r);
        base[r] = upto;
        upto = clipped(upto, n);
        if (n > 0 && upto > frees) state[r] = 1;
    }
    if (all[2] > frees) {
        part[0] = mine;
        count_rows();
        block_scan(part, all, sums);
    }
    upto = part[1];
    for (int r = r0; r < r1; r++) {
        const bool copy = forked(r);
        begin[r] = upto;
        upto += state[r] ? 0 : add[r];
        if (state[r]) len[r] = add[r] = 0, from[r] = -1;
        if (copy) state[r] = -1;
    }
    if (tid == 0) begin[R] = all[1];
    __syncthreads();
    // the free page of a rank
    auto free_page = [&](int rank) {
        const int th = last_below(holes, 0, threads, rank);
        int w = th * wper, left = rank - holes[th], n = __popc(open[w]);
        while (left >= n) {
            left -= n;
            n = __popc(open[++w]);
        }
        unsigned x = open[w];
        for (; left > 0; left--) x &= x - 1;
        return w * 32 + __ffs(x) - 1;
    };
    // a row's j-th page: kept, or new
    auto page_at = [&](int r, int j) {
        const int copied = kept(r) - (state[r] < 0 ? 1 : 0);
        return j < copied ? table[(size_t)from[r] * M + j] : free_page(base[r] + j - copied);
    };
    const int rows_per = (R + p.split - 1) / p.split, mine0 = min(R, vb * rows_per), mine1 = min(R, mine0 + rows_per);
    for (int r = mine0 + warp; r < mine1; r += warps) {
        const int total = page_of(p, len[r] + add[r] + S - 1), copied = kept(r) - (state[r] < 0 ? 1 : 0);
        const int* ids = table + (size_t)max(from[r], 0) * M;
        int* to = table_out + (size_t)r * M;
#pragma unroll 1
        for (int j0 = lane; j0 < M; j0 += 256) {
            int id[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int j = j0 + 32 * i;
                id[i] = j < copied ? ids[j] : -1;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int j = j0 + 32 * i;
                if (j < M && (j < copied || j >= total)) to[j] = id[i];
            }
        }
        for (int j = copied + lane; j < total; j += 32) to[j] = free_page(base[r] + j - copied);
    }
    for (int r = mine0 + tid; r < mine1; r += threads) {
        lens_out[r] = len[r] + add[r];
        start_out[r] = begin[r];
        status_out[r] = max(state[r], 0);
        if (f) {
            const int k = kept(r);
            fork_out[r] = state[r] < 0 ? make_int4(table[(size_t)from[r] * M + k - 1], page_at(r, k - 1), len[r] - (k - 1) * S, 0) : make_int4(-1, -1, 0, 0);
        }
    }
    if (vb == 0 && tid == 0) start_out[R] = begin[R];
    for (int i = vb * threads + tid; i < p.tokens; i += p.split * threads) {
        int4 x = make_int4(-1, -1, 0, 0);
        if (i < begin[R]) {
            const int r = last_below(begin, 0, R, i), pos = len[r] + i - begin[r], j = page_of(p, pos);
            x = make_int4(page_at(r, j) * S + pos - j * S, r, pos + 1, 0);
        }
        tok_out[i] = x;
    }
    return true;
}

// ---- append --------------------------------------------------------------------------------------------------------------
// args: k, v, tok, [fork], k_cache, v_cache.  cache[slot / ps][head][slot % ps][:] = k[token][head][:], rounded to the cache's type
// (to nearest even: the type is the caller's choice); tokens without a slot are passed over.  A fork (src, dst, n) copies the
// first n tokens of a page; new tokens are written behind them, and src's first n are written by nobody, so the order of the
// two does not matter and a second run gives the same.  Every byte is moved once, 16 at a time, eight loads of a thread under
// way: 8192 tokens of 8 heads of 128 into bf16, 100 MB, 21.0 us (0.74 of the measured copy rate: 2048 blocks of one batch of loads each, five
// to an SM, are 2.8 rounds, each with a start and an end in which little moves), 128 beams with 40 forks 4.1.
constexpr int kAppendPerBlock = 4 * kThreads * 4;       // fp32 values of k, and of v
__host__ inline int append_token_blocks(const PagedP& p) {
    return (int)(((long long)p.tokens * p.kvh * p.d + kAppendPerBlock - 1) / kAppendPerBlock);
}
// A fork's page is copied in pieces of 8 KB, a warp to one of keys or values: one warp for a whole page of 64 KB took 65 us.
constexpr int kForkPiece = 8192;
__host__ __device__ inline int append_fork_pieces(const PagedP& p) {
    return (p.ps * p.d * (p.kt == KT_FP32 ? 4 : 2) + kForkPiece - 1) / kForkPiece;
}
__host__ inline long long append_fork_blocks(const PagedP& p) {
    return p.has_fork ? ((long long)p.rows * p.kvh * append_fork_pieces(p) + 3) / 4 : 0;
}

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
    const int row4 = p.kvh * p.d >> 2, total = p.tokens * row4, shift = 31 - __clz(p.d);     // (below 2^31: the plan sees to it)
    // the loads do not wait for the slots
    float4 a[4], b[4];
    int token[4], c[4];
#pragma unroll
    for (int it = 0; it < 4; it++) {
        const int i = vb * (kAppendPerBlock / 4) + it * kThreads + threadIdx.x;
        token[it] = -1;
        if (i >= total) continue;
        token[it] = (int)((unsigned)i / (unsigned)row4);
        c[it] = (i - token[it] * row4) << 2;
        a[it] = *reinterpret_cast<const float4*>(k + (size_t)token[it] * p.qs + c[it]);
        b[it] = *reinterpret_cast<const float4*>(v + (size_t)token[it] * p.vs + c[it]);
    }
#pragma unroll
    for (int it = 0; it < 4; it++) {
        const int slot = token[it] >= 0 ? tok[token[it]].x : -1;
        if (slot < 0 || slot >= p.pages * p.ps) continue;
        const int page = page_of(p, slot), h = c[it] >> shift, e = c[it] & (p.d - 1);
        const size_t at = (((size_t)page * p.kvh + h) * p.ps + (slot - page * p.ps)) * p.d + e;
        store4(kc + at, a[it]);
        store4(vc + at, b[it]);
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
    // forks: two warps to a piece of a head's forked page, one for keys and one for values
    const int4* fork = (const int4*)t.a[3];
    const int pieces = append_fork_pieces(p), item = (vb - p.split) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 31;
    const int of = item / pieces, r = of / p.kvh, h = of - r * p.kvh;
    if (r >= p.rows) return true;
    const int4 c = fork[r];
    if ((unsigned)c.x >= (unsigned)p.pages || (unsigned)c.y >= (unsigned)p.pages || c.x == c.y) return true;
    const int e = p.kt == KT_FP32 ? 4 : 2, from = (item - of * pieces) * (kForkPiece / 16);
    const int words = min(min(c.z, p.ps) * (p.d * e / 16), from + kForkPiece / 16);
    const size_t page = (size_t)p.ps * p.d * e;
    char* cache = (char*)t.a[threadIdx.x & 32 ? 5 : 4];
    const uint4* src = (const uint4*)(cache + ((size_t)c.x * p.kvh + h) * page);
    uint4* dst = (uint4*)(cache + ((size_t)c.y * p.kvh + h) * page);
    for (int i = from + lane; i < words; i += 32 * 8) {
        uint4 x[8];
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (i + 32 * k < words) x[k] = src[i + 32 * k];
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (i + 32 * k < words) dst[i + 32 * k] = x[k];
    }
    return true;
}

}  // namespace reef
