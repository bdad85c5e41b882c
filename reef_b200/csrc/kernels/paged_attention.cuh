// Attention of one new token over a paged key-value cache [page][key head][slot][dimension]:
//   out[t][h] = sum_j p_j v_j,  p = softmax_j(q[t][h] . k_j / sqrt(d)),  j < length of token t,
// the keys of positions whose page id lies outside the cache left out; zeros where nothing is left.  (The reference attends within
// a sequence only, resource/bert/bert.cu:22-157.)
#pragma once
#include "paged_cache.cuh"

namespace reef {

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes past L1 (a cache is read once); zeros where there is nothing to read.  Volatile: it stays behind the wait for the previous
// kernel, which may have written the cache.
__device__ __forceinline__ uint4 load16(const void* at, bool there) {
    uint4 x;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                 "@p ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "=&r"(x.x), "=&r"(x.y), "=&r"(x.z), "=&r"(x.w) : "l"(at), "r"((int)there));
    return x;
}
__device__ __forceinline__ void unpack(uint4 x, float (&y)[4], float) {
    y[0] = __uint_as_float(x.x); y[1] = __uint_as_float(x.y); y[2] = __uint_as_float(x.z); y[3] = __uint_as_float(x.w);
}
__device__ __forceinline__ void unpack(uint4 x, float (&y)[8], __nv_bfloat16) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        y[2 * i] = __uint_as_float(w[i] << 16);
        y[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(uint4 x, float (&y)[8], __half) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        y[2 * i] = f.x;
        y[2 * i + 1] = f.y;
    }
}

// length of a token of the batch as far as it can be true: what a preempted kernel left behind may be anything
__device__ __forceinline__ int paged_length(const PagedP& p, int4 tok) {
    return (unsigned)tok.y < (unsigned)p.rows && tok.z > 0 ? min(tok.z, p.mp * p.ps) : 0;
}

// Where a pass over keys ends up: a warp's sums over a range of one row's keys for up to GB query heads of one key head.
// Partial results travel as [head][d + 4]: sums over the values, then the maximum (of score * log2 e) and the sum of the probabilities.
__host__ __device__ inline int paged_stride(int d) { return d + 4; }

// ---- fp32 instructions ----------------------------------------------------------------------------------------------------
// A lane holds 16 bytes of a key (4 or 8 dimensions; 8 of 256 in fp32 take two loads), the lanes of a key meet in shuffles; every
// group of lanes keeps its own maximum and sums until the end of its range.
template <class C, int D, int GB_>
struct PagedSimt {
    typedef C Cache;
    static constexpr int GB = GB_, DIM = D;
    static constexpr int VEC = 16 / (int)sizeof(C);                     // values of a load
    static constexpr int LPT = D / VEC > 32 ? 32 : D / VEC;             // lanes of a key
    static constexpr int LD = D / (VEC * LPT);                          // loads of a lane and key
    static constexpr int E = VEC * LD;                                  // dimensions of a lane
    static constexpr int TPI = 32 / LPT;                                // keys of a warp's load
    static constexpr int U = LD == 2 ? 2 : 4;                           // loads in a step
    static constexpr int UNIT = TPI * U;                                // keys of a step
    float q[GB][E], o[GB][E], m[GB], l[GB];

    static __device__ __forceinline__ int dim(int lane, int e) { return (e / VEC) * (LPT * VEC) + (lane % LPT) * VEC + e % VEC; }

    // false: the preempt flag went up
    __device__ __forceinline__ bool run(const PagedP& p, const KTask& t, int token, int row, int kh, int h0, int heads, int begin, int end, const int* flag) {
        const int lane = threadIdx.x & 31, sub = lane / LPT;
        const float scale = rsqrtf((float)D) * kLog2e;
        const float* qg = (const float*)t.a[0] + (size_t)token * p.qs + p.qo + (size_t)h0 * D;
#pragma unroll
        for (int j = 0; j < GB; j++) {
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (j < heads) x = *reinterpret_cast<const float4*>(qg + j * D + dim(lane, e));
                q[j][e] = x.x * scale; q[j][e + 1] = x.y * scale; q[j][e + 2] = x.z * scale; q[j][e + 3] = x.w * scale;
            }
#pragma unroll
            for (int e = 0; e < E; e++) o[j][e] = 0.f;
            m[j] = -INFINITY;
            l[j] = 0.f;
        }
        const int* ids = (const int*)t.a[3] + (size_t)row * p.mp;
        const C* kc = (const C*)t.a[1] + (size_t)kh * p.ps * D + (lane % LPT) * VEC;
        const C* vc = (const C*)t.a[2] + (size_t)kh * p.ps * D + (lane % LPT) * VEC;
        const size_t page = (size_t)p.kvh * p.ps * D;
        uint4 k[U][LD], v[U][LD];
        size_t at[U];
        bool there[U], next[U];
        auto find = [&](int pos0) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int pos = pos0 + u * TPI + sub;
                next[u] = pos < end;
                if (next[u]) {
                    const int j = page_of(p, pos), id = ids[j];
                    next[u] = (unsigned)id < (unsigned)p.pages;
                    at[u] = (size_t)id * page + (size_t)(pos - j * p.ps) * D;
                }
            }
        };
        auto load = [&](uint4 (&x)[U][LD], const C* from) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < LD; i++) x[u][i] = load16(from + (next[u] ? at[u] : 0) + i * LPT * VEC, next[u]);
        };
        find(begin);
        load(k, kc);
        load(v, vc);
        int up = 0, steps = 0;
#pragma unroll 1
        for (int pos = begin; pos < end; pos += UNIT) {
            if (flag != nullptr && (++steps & 7) == 0) {
                if (__any_sync(0xffffffffu, up)) return false;
                up = ld_flag(flag);
            }
#pragma unroll
            for (int u = 0; u < U; u++) there[u] = next[u];
            float s[U][GB];
#pragma unroll
            for (int u = 0; u < U; u++) {
#pragma unroll
                for (int j = 0; j < GB; j++) s[u][j] = 0.f;
#pragma unroll
                for (int i = 0; i < LD; i++) {
                    float x[VEC];
                    unpack(k[u][i], x, C());
#pragma unroll
                    for (int e = 0; e < VEC; e++)
#pragma unroll
                        for (int j = 0; j < GB; j++) s[u][j] = fmaf(q[j][i * VEC + e], x[e], s[u][j]);
                }
            }
            find(pos + UNIT);
            load(k, kc);
#pragma unroll
            for (int r = LPT / 2; r > 0; r >>= 1)
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int j = 0; j < GB; j++) s[u][j] += __shfl_xor_sync(0xffffffffu, s[u][j], r);
#pragma unroll
            for (int j = 0; j < GB; j++) {
                float top = m[j];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (!there[u]) s[u][j] = -INFINITY;
                    top = fmaxf(top, s[u][j]);
                }
                if (top != m[j]) {
                    const float by = exp2_fast(m[j] - top);
                    l[j] *= by;
#pragma unroll
                    for (int e = 0; e < E; e++) o[j][e] *= by;
                    m[j] = top;
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    s[u][j] = s[u][j] == -INFINITY ? 0.f : exp2_fast(s[u][j] - top);
                    l[j] += s[u][j];
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < LD; i++) {
                    float x[VEC];
                    unpack(v[u][i], x, C());
#pragma unroll
                    for (int e = 0; e < VEC; e++)
#pragma unroll
                        for (int j = 0; j < GB; j++) o[j][i * VEC + e] = fmaf(s[u][j], x[e], o[j][i * VEC + e]);
                }
            load(v, vc);
        }
        // the groups of lanes meet
#pragma unroll
        for (int r = LPT; r < 32; r <<= 1)
#pragma unroll
            for (int j = 0; j < GB; j++) {
                const float mo = __shfl_xor_sync(0xffffffffu, m[j], r), top = fmaxf(m[j], mo);
                const float a = m[j] == top ? 1.f : exp2_fast(m[j] - top), b = mo == top ? 1.f : exp2_fast(mo - top);
                l[j] = l[j] * a + __shfl_xor_sync(0xffffffffu, l[j], r) * b;
#pragma unroll
                for (int e = 0; e < E; e++) o[j][e] = o[j][e] * a + __shfl_xor_sync(0xffffffffu, o[j][e], r) * b;
                m[j] = top;
            }
        return true;
    }
    __device__ __forceinline__ void store(float* at, int stride, int heads, bool finished) const {
        const int lane = threadIdx.x & 31;
        if (lane >= LPT) return;
#pragma unroll
        for (int j = 0; j < GB; j++) {
            if (j >= heads) break;
            const float by = !finished ? 1.f : l[j] == 0.f ? 0.f : 1.f / l[j];
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<float4*>(at + j * stride + dim(lane, e)) = make_float4(o[j][e] * by, o[j][e + 1] * by, o[j][e + 2] * by, o[j][e + 3] * by);
            if (!finished && lane == 0) *reinterpret_cast<float2*>(at + j * stride + D) = make_float2(m[j], l[j]);
        }
    }
};

// ---- division of the work -------------------------------------------------------------------------------------------------
// Two forms.  Without parts (wpp > 0): a pass over one row's keys belongs to wpp warps of one block.  With parts (wpp = 0): the keys of
// all rows together, in units of a warp's step, are divided among all warps of the grid in equal consecutive ranges, whatever the
// rows' lengths; a pass that several blocks share leaves a part per block, which reef_paged_attention_join brings together in the
// order of the keys: no block waits for another and nothing depends on which one comes first.
constexpr int kPagedMinUnits = 2;        // units of a warp at least, before further warps take part
struct PagedSlots {
    int pair[16];                        // pass of a warp's first and last, unfinished range; -1: none
    int ends[16];                        // 1: the range begins the pass, 2: it ends it
    long long where[9];                  // first unit of every warp
    int token[8];                        // the token it lies in
    long long before[8];                 // units of the tokens before that one
    long long sums[8];
};
template <class E>
__device__ __forceinline__ bool paged_attention_body(const KTask& t, int vb, unsigned char* smem, const int* flag) {
    const PagedP& p = t.p.paged;
    const int4* tok = (const int4*)t.a[4];
    float* out = (float*)t.a[5];
    PagedSlots& sl = *reinterpret_cast<PagedSlots*>(smem);
    float* slot = reinterpret_cast<float*>(smem + ((sizeof(PagedSlots) + 15) & ~15));
    const int stride = paged_stride(E::DIM), slot_floats = E::GB * stride;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x;
    const int P = p.kvh * p.subs, group = p.heads / p.kvh;
    __syncthreads();                     // a persistent caller's previous block is out of shared memory
    if (tid < 16) sl.pair[tid] = -1;
    bool stopped = false;
    E e;
    auto where_out = [&](int pair, int* heads) {
        const int token = pair / P, r = pair - token * P, kh = r / p.subs, h0 = kh * group + (r - kh * p.subs) * E::GB;
        *heads = min(E::GB, (kh + 1) * group - h0);
        return out + ((size_t)token * p.heads + h0) * E::DIM;
    };
    // units [a, b) of a pass of n
    auto range = [&](int token, int r, int4 tk, int a, int b, int n, int s) {
        const int kh = r / p.subs, h0 = kh * group + (r - kh * p.subs) * E::GB, heads = min(E::GB, (kh + 1) * group - h0);
        if (!e.run(p, t, token, tk.y, kh, h0, heads, a * E::UNIT, min(b * E::UNIT, paged_length(p, tk)), flag)) return false;
        if (a == 0 && b == n) {
            e.store(out + ((size_t)token * p.heads + h0) * E::DIM, E::DIM, heads, true);
        } else {
            e.store(slot + s * slot_floats, stride, heads, false);
            if (lane == 0) {
                sl.pair[s] = token * P + r;
                sl.ends[s] = (a == 0 ? 1 : 0) | (b == n ? 2 : 0);
            }
        }
        return true;
    };
    if (p.wpp > 0) {
        const long long pair = (long long)vb * (8 / p.wpp) + warp / p.wpp;
        __syncthreads();
        if (pair < (long long)p.tokens * P) {
            const int token = (int)(pair / P), i = warp % p.wpp;
            const int4 tk = tok[token];
            const int n = (paged_length(p, tk) + E::UNIT - 1) / E::UNIT;
            const int a = (int)((long long)n * i / p.wpp), b = (int)((long long)n * (i + 1) / p.wpp);
            if (a < b) stopped = !range(token, (int)(pair - (long long)token * P), tk, a, b, n, 2 * warp + (a == 0 ? 1 : 0));
            if (n == 0 && i == 0) {
                int heads;
                float* at = where_out((int)pair, &heads);
                for (int c = lane * 4; c < heads * E::DIM; c += 128) *reinterpret_cast<float4*>(at + c) = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    } else {
        // units of the tokens, a run of tokens to a thread
        const int per = (p.tokens + kThreads - 1) / kThreads, t0 = min(p.tokens, tid * per), t1 = min(p.tokens, t0 + per);
        long long mine = 0;
        for (int i = t0; i < t1; i++) mine += (paged_length(p, tok[i]) + E::UNIT - 1) / E::UNIT;
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        if (lane == 31) sl.sums[warp] = upto;
        __syncthreads();
        long long all = 0, before = 0;
#pragma unroll
        for (int w = 0; w < 8; w++) {
            if (w < warp) before += sl.sums[w];
            all += sl.sums[w];
        }
        upto += before;
        const long long W = all * P;
        const int blocks = (int)min((long long)t.nblocks, (W + 8 * kPagedMinUnits - 1) / (8 * kPagedMinUnits));
        const long long lo = vb < blocks ? W * vb / blocks : W, hi = vb < blocks ? W * (vb + 1) / blocks : W;
        for (int w = 0; w < 8; w++) {
            const long long at = lo + (hi - lo) * w / 8, ex = (upto - mine) * P;
            if (tid == 0) {
                sl.where[w] = at;
                if (w == 0) sl.where[8] = hi;
            }
            if (at < hi && at >= ex && at < upto * P) {
                long long b = upto - mine;
                int i = t0;
                for (; i < t1; i++) {
                    const int n = (paged_length(p, tok[i]) + E::UNIT - 1) / E::UNIT;
                    if (at < (b + n) * P) break;
                    b += n;
                }
                sl.token[w] = i;
                sl.before[w] = b;
            }
        }
        __syncthreads();
        long long u = sl.where[warp];
        const long long end = sl.where[warp + 1];
        if (u < end) {
            int token = sl.token[warp];
            long long base = sl.before[warp] * P;      // units before this token
            while (u < end && token < p.tokens) {
                const int4 tk = tok[token];
                const int n = (paged_length(p, tk) + E::UNIT - 1) / E::UNIT;
                if (u >= base + (long long)n * P) {
                    base += (long long)n * P;
                    token++;
                    continue;
                }
                const int r = (int)((u - base) / n), a = (int)(u - base - (long long)r * n), b = (int)min((long long)n, a + (end - u));
                if (!range(token, r, tk, a, b, n, 2 * warp + (a == 0 ? 1 : 0))) {
                    stopped = true;
                    break;
                }
                u += b - a;
            }
        }
        // rows without keys
        for (int i = vb; i < p.tokens; i += t.nblocks)
            if (paged_length(p, tok[i]) == 0)
                for (int c = tid * 4; c < p.heads * E::DIM; c += kThreads * 4) *reinterpret_cast<float4*>(out + (size_t)i * p.heads * E::DIM + c) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (__syncthreads_or(stopped)) return false;
    // ranges of one pass that lie side by side, joined by the warp that has the first of them
    if (p.wpp == 0 && tid < 2) {
        int* desc = (int*)t.a[6] + 2 * vb;
        // what this block leaves: a pass that began earlier (0), one that goes on behind it (1)
        int got = -1;
        if (tid == 0) {
            int i = 0;
            while (i < 16 && sl.pair[i] < 0) i++;
            if (i < 16 && !(sl.ends[i] & 1)) got = sl.pair[i];
        } else {
            int i = 15, j;
            while (i >= 0 && sl.pair[i] < 0) i--;
            if (i >= 0 && !(sl.ends[i] & 2)) {
                for (j = i; j >= 0 && (sl.pair[j] < 0 || sl.pair[j] == sl.pair[i]); j--)
                    if (sl.pair[j] == sl.pair[i] && (sl.ends[j] & 1)) got = sl.pair[i];
            }
        }
        desc[tid] = got;
    }
    for (int s = 2 * warp; s < 2 * warp + 2; s++) {
        const int pair = sl.pair[s];
        if (pair < 0) continue;
        bool first = true;
        for (int i = s - 1; i >= 0; i--)
            if (sl.pair[i] >= 0) {
                first = sl.pair[i] != pair;
                break;
            }
        if (!first) continue;
        unsigned chain = 1u << s;
        int ends = sl.ends[s];
        for (int i = s + 1; i < 16; i++) {
            if (sl.pair[i] < 0) continue;
            if (sl.pair[i] != pair) break;
            chain |= 1u << i;
            ends |= sl.ends[i];
        }
        int heads;
        float* at = where_out(pair, &heads);
        const bool whole = ends == 3;
        int step = E::DIM;
        if (!whole) {
            // (only with parts)
            at = (float*)t.a[6] + 2 * ((t.nblocks + 1) & ~1) + ((size_t)vb * 2 + (ends & 1)) * slot_floats;
            step = stride;
        }
        for (int j = 0; j < heads; j++) {
            float top = -INFINITY, sum = 0.f;
            for (unsigned c = chain; c; c &= c - 1) top = fmaxf(top, slot[(__ffs(c) - 1) * slot_floats + j * stride + E::DIM]);
            float4 o[(E::DIM + 127) / 128];
#pragma unroll
            for (int x = 0; x < (E::DIM + 127) / 128; x++) o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (unsigned c = chain; c; c &= c - 1) {
                const float* from = slot + (__ffs(c) - 1) * slot_floats + j * stride;
                const float by = from[E::DIM] == top ? 1.f : exp2_fast(from[E::DIM] - top);
                sum = fmaf(from[E::DIM + 1], by, sum);
#pragma unroll
                for (int x = 0; x < (E::DIM + 127) / 128; x++)
                    if (x * 128 + lane * 4 < E::DIM) {
                        const float4 y = *reinterpret_cast<const float4*>(from + x * 128 + lane * 4);
                        o[x].x = fmaf(y.x, by, o[x].x); o[x].y = fmaf(y.y, by, o[x].y); o[x].z = fmaf(y.z, by, o[x].z); o[x].w = fmaf(y.w, by, o[x].w);
                    }
            }
            const float by = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int x = 0; x < (E::DIM + 127) / 128; x++)
                if (x * 128 + lane * 4 < E::DIM)
                    *reinterpret_cast<float4*>(at + (size_t)j * step + x * 128 + lane * 4) = make_float4(o[x].x * by, o[x].y * by, o[x].z * by, o[x].w * by);
            if (!whole && lane == 0) *reinterpret_cast<float2*>(at + (size_t)j * step + E::DIM) = make_float2(top, sum);
        }
    }
    return true;
}

// ---- shapes ---------------------------------------------------------------------------------------------------------------
__host__ inline int paged_gb_max(int kt, int) { return kt == KT_FP32 ? 4 : 2; }
__host__ inline int paged_unit(const PagedP& p) {          // keys of a warp's step (UNIT above)
    const int vec = p.kt == KT_FP32 ? 4 : 8, lanes = p.d / vec > 32 ? 32 : p.d / vec;
    return 32 / lanes * (p.d > 32 * vec ? 2 : 4);
}
__host__ inline int paged_attention_smem(const PagedP& p) { return (int)((sizeof(PagedSlots) + 15) & ~15) + 16 * p.gb * paged_stride(p.d) * 4; }
__host__ inline size_t paged_parts_bytes(const PagedP& p, int blocks) {
    return ((size_t)2 * ((blocks + 1) & ~1) + (size_t)blocks * 2 * p.gb * paged_stride(p.d)) * 4;
}

constexpr int kSmsPlanned = 148;                           // launch geometry is planned without a GPU
constexpr int kPagedSmemMax = 100 * 1024;                  // two blocks to an SM
static_assert(4 * ((kTablesMaxPages + 31) / 32 + 6 * kTablesMaxRows + 34) <= kPagedSmemMax, "the largest page tables");

// ---- join -----------------------------------------------------------------------------------------------------------------
// args: parts, out.  A block per head of the pass that the vb-th block left unfinished: its part, then those of the blocks behind it
// that lie in the same pass, a share of them to every group of lanes.
__device__ __forceinline__ bool body_paged_join(const KTask& t, int vb, unsigned char* smem, const int*) {
    const PagedP& p = t.p.paged;
    const int blocks = p.split, j = vb % p.gb, b = vb / p.gb, tid = threadIdx.x, D = p.d;
    const int* desc = (const int*)t.a[0];
    const int stride = paged_stride(D), P = p.kvh * p.subs, group = p.heads / p.kvh;
    const size_t slot_floats = (size_t)p.gb * stride;
    const float* part = (const float*)t.a[0] + 2 * ((blocks + 1) & ~1) + (size_t)j * stride;
    const int pair = desc[2 * b + 1];
    if (pair < 0 || pair >= p.tokens * P) return true;
    const int token = pair / P, r = pair - token * P, kh = r / p.subs, h = kh * group + (r - kh * p.subs) * p.gb + j;
    if (h >= (kh + 1) * group) return true;
    __shared__ float red[2][8];
    __shared__ int last;
    // blocks b + 1 .. b + n - 1 lie in this pass
    __syncthreads();
    if (tid == 0) last = blocks;
    __syncthreads();
    for (int i = b + 1 + tid; i < blocks; i += kThreads)
        if (desc[2 * i] != pair) {
            atomicMin(&last, i);
            break;
        }
    __syncthreads();
    const int n = last - b;
    auto at = [&](int i) { return part + ((size_t)(b + i) * 2 + (i == 0 ? 1 : 0)) * slot_floats; };
    float top = -INFINITY;
    for (int i = tid; i < n; i += kThreads) top = fmaxf(top, at(i)[D]);
    top = warp_max(top);
    if ((tid & 31) == 0) red[0][tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = fmaxf(top, red[0][w]);
    // groups of D / 4 lanes, each with every G-th part
    const int L = D / 4, G = kThreads / L, g = tid / L, c = (tid - g * L) * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int i = g; i < n; i += G) {
        const float* x = at(i);
        const float2 ml = *reinterpret_cast<const float2*>(x + D);
        const float4 y = *reinterpret_cast<const float4*>(x + c);
        const float by = ml.x == top ? 1.f : exp2_fast(ml.x - top);
        sum = fmaf(ml.y, by, sum);
        o.x = fmaf(y.x, by, o.x); o.y = fmaf(y.y, by, o.y); o.z = fmaf(y.z, by, o.z); o.w = fmaf(y.w, by, o.w);
    }
    float* mine = reinterpret_cast<float*>(smem) + (size_t)g * stride;
    *reinterpret_cast<float4*>(mine + c) = o;
    if (c == 0) mine[D] = sum;
    __syncthreads();
    if (g == 0) {
        for (int i = 1; i < G; i++) {
            const float* x = reinterpret_cast<const float*>(smem) + (size_t)i * stride;
            const float4 y = *reinterpret_cast<const float4*>(x + c);
            o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
            sum += x[D];
        }
        const float by = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<float4*>((float*)t.a[1] + ((size_t)token * p.heads + h) * D + c) = make_float4(o.x * by, o.y * by, o.z * by, o.w * by);
    }
    return true;
}
__host__ inline int paged_join_smem(int d) { return kThreads / (d / 4) * paged_stride(d) * 4; }

}  // namespace reef
