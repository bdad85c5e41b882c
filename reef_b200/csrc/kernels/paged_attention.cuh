// Attention of one new token over a paged key-value cache [page][key head][slot][dimension]:
//   out[t][h] = sum_j p_j v_j,  p = softmax_j(q[t][h] . k_j / sqrt(d)),  j < length of token t,
// the keys of positions whose page id lies outside the cache left out; zeros where nothing is left.  (The reference attends within
// a sequence only, resource/bert/bert.cu:22-157.)
//
// One pass over the keys with a running maximum and sum; every key and value is read once for up to eight query heads (fp32 with 256
// dimensions: four), and again for every further eight: 64 rows, 292368 keys of one key head, 128 dimensions, bf16, 8 heads 43 us, 16 64, 64 205;
// 64 rows of 128 heads over 8 389, of 64 heads 227.  Bound by HBM where there is much to read: 64 rows of 32 heads over 8, bf16, 128 dimensions,
// 860 MB in 160 us with the join (5.4 TB/s, 0.83 of the measured copy rate; SMs do not get equal shares of it), 2048 passes of up to 1 MB
// 185 us (0.89); fp32 in groups of five, 2.4 GB in 413 us (0.90), 188 MB in 47 (0.62, dependent steps).  A call with little to read is a
// chain of latencies: 12 heads of a row of 77 keys 5.0 us, of 1000 14.
#pragma once
#include "bf16_split.cuh"
#include "paged_cache.cuh"

namespace reef {

// 16 bytes into shared memory, past L1 (a cache is read once); zeros where there is nothing to read
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 read16(uint32_t from) {
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(from) : "memory");
    return x;
}
__device__ __forceinline__ void unpack(uint4 x, float2 (&y)[2], float) {
    y[0] = make_float2(__uint_as_float(x.x), __uint_as_float(x.y));
    y[1] = make_float2(__uint_as_float(x.z), __uint_as_float(x.w));
}
__device__ __forceinline__ void unpack(uint4 x, float2 (&y)[4], __nv_bfloat16) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void unpack(uint4 x, float2 (&y)[4], __half) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}

// length of a token of the batch as far as it can be true: what a preempted kernel left behind may be anything
__device__ __forceinline__ int paged_length(const PagedP& p, int4 tok) {
    return (unsigned)tok.y < (unsigned)p.rows && tok.z > 0 ? min(tok.z, p.mp * p.ps) : 0;
}

// Where a pass over keys ends up: a warp's sums over a range of one row's keys for up to GB query heads of one key head.
// Partial results travel as [head][d + 4]: sums over the values, then the maximum (of score * log2 e) and the sum of the probabilities.
__host__ __device__ constexpr int paged_stride(int d) { return d + 4; }

// What a pass looks at: the queries that share it, one row's pages, one key head of the cache.
struct PagedRow {
    const float* q;           // first query head
    const char *k, *v;        // caches
    const int* ids;
    int heads, begin, end;    // query heads; keys [begin, end)
    int ps, pages, kvh, kh;
    unsigned ps_mul;
    int ps_shift;
    // page of a key, asked for a step ahead of its use
    __device__ __forceinline__ int page(int pos) const { return pos < end ? ids[__umulhi((unsigned)pos << 1, ps_mul) >> ps_shift] : -1; }
    // place of a key among the keys of all pages and heads, -1 for none (fewer than 2^31: the plan sees to it)
    __device__ __forceinline__ int place(int pos, int id) const {
        const int j = (int)(__umulhi((unsigned)pos << 1, ps_mul) >> ps_shift);
        return (unsigned)id < (unsigned)pages ? (id * kvh + kh) * ps + (pos - j * ps) : -1;
    }
};

// How keys and values reach a warp: a step's keys, its values, the next step's keys ... go through a ring of RING stages of its own in
// shared memory by cp.async, RING - 1 of them under way.  A warp's request covers 512 bytes that lie together in memory: lanes that fetched
// the pieces they use themselves, 32 bytes of every row, had half of the bandwidth (3.7 instead of 6.8 TB/s from tiles of 4 KB).
// Stages of a ring: as many as the blocks of an SM find room for, two with fp32 instructions, one on the tensor cores.  There the operands do
// not fit 128 registers, and fewer warps with more under way each leave fewer parts and less to join: a row of 131072 keys 34 and 8 us with two
// blocks to an SM and 3 stages, 30 and 6 with one block and 6; 90 rows of 48 heads over 6 75 and 65, of 24 heads 58 and 59.
constexpr int kPagedSimtRing = 6;
__host__ __device__ constexpr int paged_mma_ring(int d) { return 768 / d; }
// (a range that is worked out again needs its slot and a ring of its own)
__host__ __device__ constexpr int paged_mma_scratch(int d, int heads) {
    const int ring = paged_mma_ring(d) * d * 32, again = heads * paged_stride(d) * 4 + 4 * 2048;
    return ring > again ? ring : again;
}
template <int RING, int BYTES>
struct PagedRing {
    uint32_t base, in, out;
    __device__ __forceinline__ PagedRing(char* at) {
        in = out = base = (uint32_t)__cvta_generic_to_shared(at);
    }
    __device__ __forceinline__ uint32_t put() {
        const uint32_t at = in;
        in = in == base + (RING - 1) * BYTES ? base : in + BYTES;
        return at;
    }
    __device__ __forceinline__ uint32_t take() {
        copy_wait<RING - 2>();
        const uint32_t at = out;
        out = out == base + (RING - 1) * BYTES ? base : out + BYTES;
        return at;
    }
};

// ---- fp32 instructions ----------------------------------------------------------------------------------------------------
// A lane holds 16 bytes of a key (4 or 8 dimensions; 8 of 256 in fp32 take two pieces).  The lanes of a key bring their parts of the scores
// together by halves, so that in the end every score stands in a lane of its own: half as many shuffles as sums over all lanes, and one
// exponential for all scores of a step instead of one each.  Every group of lanes keeps its own maximum and sums until the end of its range.
__host__ __device__ constexpr int paged_log2(int x) { return x <= 1 ? 0 : 1 + paged_log2(x / 2); }
__host__ __device__ constexpr int paged_pow2(int x) { return x <= 1 ? 1 : 2 * paged_pow2((x + 1) / 2); }
// keys of a lane in a step: its scores fill at most the lanes of a key, and registers
__host__ __device__ constexpr int paged_simt_keys(int pieces, int lanes, int gb) {
    const int most = (gb > 6 ? 2 : 4) / pieces, room = lanes / paged_pow2(gb);
    return most < room ? most : room;
}
template <class C, int D, int GB_, int RING_ = kPagedSimtRing>
struct PagedSimt {
    static constexpr int GB = GB_, DIM = D, RING = RING_;
    static constexpr int VEC = 16 / (int)sizeof(C);                     // values of a piece
    static constexpr int LPT = D / VEC > 32 ? 32 : D / VEC;             // lanes of a key
    static constexpr int LD = D / (VEC * LPT);                          // pieces of a lane and key
    static constexpr int E = VEC * LD;                                  // dimensions of a lane
    static constexpr int TPI = 32 / LPT;                                // keys of a warp's piece
    static constexpr int U = paged_simt_keys(LD, LPT, GB);              // keys of a lane in a step
    static constexpr int UNIT = TPI * U;                                // keys of a step
    static constexpr int STAGE = U * LD * 512, SCRATCH = RING * STAGE > GB * paged_stride(D) * 4 ? RING * STAGE : GB * paged_stride(D) * 4;
    static constexpr int G2 = paged_pow2(GB), N = U * G2, SPREAD = LPT / N;     // scores of a step and key lane; lanes that hold the same one
    static_assert(N <= LPT, "a lane to a score");
    float2 q[GB][E / 2], o[GB][E / 2];
    float m, l;                                                          // of this lane's head

    static __device__ __forceinline__ int dim(int lane, int e) { return (e / VEC) * (LPT * VEC) + (lane % LPT) * VEC + e % VEC; }
    // the lane (of this lane's group) that has the score of its u-th key and head j
    static __device__ __forceinline__ int holder(int lane, int u, int j) { return lane / LPT * LPT + (u * G2 + j) * SPREAD; }

    // false: the preempt flag went up
    __device__ __forceinline__ bool run(const PagedRow& r, char* scratch, const int* flag) {
        const int lane = threadIdx.x & 31, sub = lane / LPT, mine_u = lane % LPT / SPREAD / G2;
        const C* kc = (const C*)r.k + (lane % LPT) * VEC;
        const C* vc = (const C*)r.v + (lane % LPT) * VEC;
        PagedRing<RING, STAGE> ring(scratch + lane * 16);        // (a lane's pieces are its own)
        // a step's keys lie in one page where the pages hold whole steps (steps begin at multiples of their size)
        const bool one_page = r.ps % UNIT == 0;
        int at[U], id[U], pos_in = r.begin;
#pragma unroll
        for (int u = 0; u < U; u++) at[u] = -1, id[u] = r.page(r.begin + u * TPI + sub);
        unsigned there = 0;             // a bit per key of a lane, four to a step, the newest lowest
        auto issue_k = [&]() {
            const uint32_t to = ring.put();
            there <<= 4;
            if (pos_in < r.end) {
                if (one_page) {
                    at[0] = r.place(pos_in + sub, __shfl_sync(0xffffffffu, id[0], 0));   // (the first key is there)
#pragma unroll
                    for (int u = 1; u < U; u++) at[u] = at[0] >= 0 && pos_in + u * TPI + sub < r.end ? at[0] + u * TPI : -1;
                    if (pos_in + sub >= r.end) at[0] = -1;
                    id[0] = r.page(pos_in + UNIT);
                } else {
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        at[u] = r.place(pos_in + u * TPI + sub, id[u]);
                        id[u] = r.page(pos_in + UNIT + u * TPI + sub);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    there |= (at[u] >= 0 ? 1u : 0u) << u;
                    const C* from = kc + (size_t)max(at[u], 0) * D;
#pragma unroll
                    for (int i = 0; i < LD; i++) copy16(to + (u * LD + i) * 512, from + i * LPT * VEC, at[u] >= 0);
                }
            }
            copy_commit();
        };
        auto issue_v = [&]() {
            const uint32_t to = ring.put();
            if (pos_in < r.end) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const C* from = vc + (size_t)max(at[u], 0) * D;
#pragma unroll
                    for (int i = 0; i < LD; i++) copy16(to + (u * LD + i) * 512, from + i * LPT * VEC, at[u] >= 0);
                }
            }
            copy_commit();
            pos_in += UNIT;
        };
        static_assert(RING % 2 == 0, "a ring begins with keys and ends with keys under way");
        issue_k();
#pragma unroll
        for (int i = 0; i < RING / 2 - 1; i++) {
            issue_v();
            issue_k();
        }
        const float scale = rsqrtf((float)D) * kLog2e;
#pragma unroll
        for (int j = 0; j < GB; j++) {
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (j < r.heads) x = *reinterpret_cast<const float4*>(r.q + j * D + dim(lane, e));
                q[j][e / 2] = make_float2(x.x * scale, x.y * scale);
                q[j][e / 2 + 1] = make_float2(x.z * scale, x.w * scale);
            }
#pragma unroll
            for (int e = 0; e < E / 2; e++) o[j][e] = make_float2(0.f, 0.f);
        }
        m = -INFINITY;
        l = 0.f;
        int up = 0, steps = 0;
        bool stopped = false;
#pragma unroll 1
        for (int pos = r.begin; pos < r.end; pos += UNIT) {
            if (flag != nullptr && (++steps & 7) == 0) {
                if (__any_sync(0xffffffffu, up)) {
                    stopped = true;
                    break;
                }
                up = ld_flag(flag);
            }
            uint32_t from = ring.take();
            float s[N];
#pragma unroll
            for (int u = 0; u < U; u++) {
                float2 sum[GB];
#pragma unroll
                for (int j = 0; j < GB; j++) sum[j] = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < LD; i++) {
                    float2 y[VEC / 2];
                    unpack(read16(from + (u * LD + i) * 512), y, C());
#pragma unroll
                    for (int e = 0; e < VEC / 2; e++)
#pragma unroll
                        for (int j = 0; j < GB; j++) sum[j] = fma2(q[j][i * VEC / 2 + e], y[e], sum[j]);
                }
#pragma unroll
                for (int j = 0; j < G2; j++) s[u * G2 + j] = j < GB ? sum[j < GB ? j : 0].x + sum[j < GB ? j : 0].y : 0.f;
            }
            issue_v();
            const unsigned now = there >> (RING - 1) / 2 * 4;            // (as many steps are ahead of this one)
            // a lane keeps the half of the scores that its bit names and gives the other one away
#pragma unroll
            for (int level = 1; level <= paged_log2(LPT); level++) {
                const int w = LPT >> level, n = N >> level;
                if (n > 0) {
                    const bool upper = lane & w;
#pragma unroll
                    for (int i = 0; i < N / 2; i++) {
                        if (i >= n) break;
                        const float give = upper ? s[i] : s[n + i];
                        s[i] = (upper ? s[n + i] : s[i]) + __shfl_xor_sync(0xffffffffu, give, w);
                    }
                } else {
                    s[0] += __shfl_xor_sync(0xffffffffu, s[0], w);
                }
            }
            const float score = now >> mine_u & 1 ? s[0] : -INFINITY;
            float top = fmaxf(m, score);
#pragma unroll
            for (int w = LPT / U; w < LPT; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            if (__any_sync(0xffffffffu, top != m)) {
                const float by = top == m ? 1.f : exp2_fast(m - top);
                l *= by;
#pragma unroll
                for (int j = 0; j < GB; j++) {
                    const float b = __shfl_sync(0xffffffffu, by, holder(lane, 0, j));
#pragma unroll
                    for (int e = 0; e < E / 2; e++) o[j][e] = make_float2(o[j][e].x * b, o[j][e].y * b);
                }
                m = top;
            }
            const float p = score == -INFINITY ? 0.f : exp2_fast(score - top);
            l += p;
            from = ring.take();
#pragma unroll
            for (int u = 0; u < U; u++) {
                float2 y[E / 2];
#pragma unroll
                for (int i = 0; i < LD; i++) {
                    float2 z[VEC / 2];
                    unpack(read16(from + (u * LD + i) * 512), z, C());
#pragma unroll
                    for (int e = 0; e < VEC / 2; e++) y[i * VEC / 2 + e] = z[e];
                }
#pragma unroll
                for (int j = 0; j < GB; j++) {
                    const float b = __shfl_sync(0xffffffffu, p, holder(lane, u, j));
#pragma unroll
                    for (int e = 0; e < E / 2; e++) o[j][e] = fma2(make_float2(b, b), y[e], o[j][e]);
                }
            }
            issue_k();
        }
        copy_wait<0>();
        if (stopped) return false;
        // the keys of a lane group's lanes, then the groups
#pragma unroll
        for (int w = LPT / U; w < LPT; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
#pragma unroll
        for (int w = LPT; w < 32; w <<= 1) {
            const float mo = __shfl_xor_sync(0xffffffffu, m, w), top = fmaxf(m, mo);
            const float a = m == top ? 1.f : exp2_fast(m - top), b = mo == top ? 1.f : exp2_fast(mo - top);
            l = l * a + __shfl_xor_sync(0xffffffffu, l, w) * b;
            m = top;
#pragma unroll
            for (int j = 0; j < GB; j++) {
                const float aj = __shfl_sync(0xffffffffu, a, holder(lane, 0, j)), bj = __shfl_sync(0xffffffffu, b, holder(lane, 0, j));
#pragma unroll
                for (int e = 0; e < E / 2; e++) {
                    o[j][e].x = o[j][e].x * aj + __shfl_xor_sync(0xffffffffu, o[j][e].x, w) * bj;
                    o[j][e].y = o[j][e].y * aj + __shfl_xor_sync(0xffffffffu, o[j][e].y, w) * bj;
                }
            }
        }
        return true;
    }
    __device__ __forceinline__ void store(const PagedRow& r, float* at, int stride, bool finished) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int j = 0; j < GB; j++) {
            const float lj = __shfl_sync(0xffffffffu, l, holder(0, 0, j)), mj = __shfl_sync(0xffffffffu, m, holder(0, 0, j));
            if (j >= r.heads || lane >= LPT) continue;
            const float by = !finished ? 1.f : lj == 0.f ? 0.f : 1.f / lj;
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<float4*>(at + j * stride + dim(lane, e)) =
                    make_float4(o[j][e / 2].x * by, o[j][e / 2].y * by, o[j][e / 2 + 1].x * by, o[j][e / 2 + 1].y * by);
            if (!finished && lane == 0) *reinterpret_cast<float2*>(at + j * stride + D) = make_float2(mj, lj);
        }
    }
};

// ---- tensor cores -----------------------------------------------------------------------------------------------------------
// From three query heads to a key head on, the multiplications of the fp32 form are what takes the time (64 rows of 32 heads over 8 as above:
// 375 us); 16-bit keys and values are operands of mma.sync as they are.  Queries and probabilities keep their 32 bits: a bf16 query is the
// exact sum of three bf16 values, an fp16 one that of two fp16 values, scaled to the type's range, but for 2^-22 of it or 2^-39 of the
// largest.  The sixteen rows of a multiplication hold four or eight heads' parts side by side, so that one instruction, or two, multiplies
// all of them.  Sums are carried on outside the tensor core, whose additions truncate.
// A warp takes 16 keys at a time, from its ring into registers in the operands' layout: lane (g, c) has 16-byte pieces of keys g and 8 + g,
// whose eight dimensions are its K positions of two instructions; and of the values of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 eight dimensions,
// which are its columns of eight instructions.  These multiplications keep the tensor pipe 19 % busy while HBM is the bound, so that the
// 128 rows of a tcgen05 tile would wait for the same bytes.
// What the parts cannot carry (an infinity or NaN among the operands) ends as a sum that is not finite: such a range is worked out again by
// fp32 instructions, as is one whose queries are of sizes that two fp16 values cannot hold side by side.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Rows of a multiplication's first operand: two values of 32 bits (K positions 2 c and 2 c + 1), as the parts that this lane's rows g and
// g + 8 hold.  bf16, four heads: h in rows 0 - 3, m in 4 - 7, l in 8 - 11.  bf16, eight heads: h in rows 0 - 7, m in 8 - 15, l in an
// instruction of its own.  fp16, eight heads: h in rows 0 - 7, m in 8 - 15.
template <class C, int HEADS> struct Rows;
template <> struct Rows<__nv_bfloat16, 4> {
    uint32_t lo, hi;
    __device__ __forceinline__ void set(float x, float y) {
        const Bf16Triple t = bf16_split(x, y);
        const bool second = threadIdx.x & 16;
        lo = second ? t.m : t.h;
        hi = second ? 0u : t.l;
    }
    static constexpr float kLift = 0.f;       // exponent added to probabilities
    static constexpr bool kScaled = false, kHalves = true;
};
template <> struct Rows<__nv_bfloat16, 8> {
    uint32_t lo, hi, l;
    __device__ __forceinline__ void set(float x, float y) {
        const Bf16Triple t = bf16_split(x, y);
        lo = t.h; hi = t.m; l = t.l;
    }
    static constexpr float kLift = 0.f;
    static constexpr bool kScaled = false, kHalves = false;
};
template <> struct Rows<__half, 8> {
    uint32_t lo, hi;
    __device__ __forceinline__ void set(float x, float y) {
        const __half2 a = __floats2half2_rn(x, y);
        const float2 f = __half22float2(a);
        const __half2 b = __floats2half2_rn(x - f.x, y - f.y);
        lo = *reinterpret_cast<const uint32_t*>(&a);
        hi = *reinterpret_cast<const uint32_t*>(&b);
    }
    // a probability of 1 becomes 2^15: two fp16 values have 22 bits of it down to 2^-18; of smaller ones 2^-40 is lost at most
    static constexpr float kLift = 15.f;
    static constexpr bool kScaled = true, kHalves = false;
};
template <> struct Rows<__half, 4> : Rows<__half, 8> {};
// d = or += the products of 16 K positions
template <int H>
__device__ __forceinline__ void mma_rows(float (&d)[4], const Rows<__nv_bfloat16, H>& a, const Rows<__nv_bfloat16, H>& b, uint32_t b0, uint32_t b1, bool first) {
    if constexpr (H == 8) {
        if (first) mma_bf16_zero(d, a.l, 0u, b.l, 0u, b0, b1);
        else mma_bf16(d, a.l, 0u, b.l, 0u, b0, b1);
        mma_bf16(d, a.lo, a.hi, b.lo, b.hi, b0, b1);
    } else {
        if (first) mma_bf16_zero(d, a.lo, a.hi, b.lo, b.hi, b0, b1);
        else mma_bf16(d, a.lo, a.hi, b.lo, b.hi, b0, b1);
    }
}
template <int H>
__device__ __forceinline__ void mma_rows(float (&d)[4], const Rows<__half, H>& a, const Rows<__half, H>& b, uint32_t b0, uint32_t b1, bool first) {
    if (first) d[0] = d[1] = d[2] = d[3] = 0.f;
    mma_f16(d, a.lo, a.hi, b.lo, b.hi, b0, b1);
}

template <class C, int D>
__device__ __noinline__ void paged_again(PagedRow r, char* scratch, float* at, int stride, bool finished) {
    const int heads = r.heads;
    r.heads = 1;
#pragma unroll 1
    for (int j = 0; j < heads; j++) {
        PagedSimt<C, D, 1, 4> e;
        e.run(r, scratch, nullptr);
        e.store(r, at + j * stride, stride, finished);
        r.q += D;
    }
}

template <class C_, int D, int HEADS>
struct PagedMma {
    typedef C_ C;
    typedef Rows<C, HEADS> A;
    static constexpr int GB = HEADS, DIM = D, UNIT = 16, KS = D / 16, RING = paged_mma_ring(D), STAGE = D * 32;
    static constexpr int SCRATCH = paged_mma_scratch(D, HEADS);
    float2 o[D / 8];                // of this lane's head: dimensions 64 (i / 8) + 16 c + i % 8 and 8 further
    float m, l;
    char* spare;
    bool lost;

    // sixteen keys (values) as they lie in memory, 512 bytes of them at a time; in shared memory the 16-byte pieces of a row change places
    // among eight, so that the pieces a quarter of a warp reads lie in different banks
    template <class Swap>
    static __device__ __forceinline__ void copy_tile(uint32_t to, const char* cache, int mine, Swap swap) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            const int byte = i * 512 + lane * 16, row = byte / (2 * D), piece = byte % (2 * D) / 16;
            const int at = __shfl_sync(0xffffffffu, mine, row);
            copy16(to + row * 2 * D + (piece ^ swap(row)) * 16, cache + (size_t)max(at, 0) * 2 * D + piece * 16, at >= 0);
        }
    }
    __device__ __forceinline__ bool run(const PagedRow& r, char* scratch, const int* flag) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, head = g & (HEADS - 1);
        spare = scratch + GB * paged_stride(D) * 4;
        PagedRing<RING, STAGE> ring(scratch);
        int mine, pos_k = r.begin, pos_v = r.begin, id = r.page(r.begin + (lane & 15));
        unsigned there = 0;             // a bit per score of a lane, four to a step, the newest lowest
        auto issue_k = [&]() {
            const uint32_t to = ring.put();
            there <<= 4;
            if (pos_k < r.end) {
                mine = r.place(pos_k + (lane & 15), id);
                id = r.page(pos_k + UNIT + (lane & 15));
                copy_tile(to, r.k, mine, [](int row) { return (row & 1) << 2; });
                const unsigned all = __ballot_sync(0xffffffffu, mine >= 0) >> 2 * c;
                there |= (all & 3) | (all >> 6 & 12);
            }
            copy_commit();
            pos_k += UNIT;
        };
        auto issue_v = [&]() {
            const uint32_t to = ring.put();
            if (pos_v < r.end) {
                copy_tile(to, r.v, mine, [](int row) { return row & 6; });
            }
            copy_commit();
            pos_v += UNIT;
        };
        issue_k();
        issue_v();
#pragma unroll
        for (int i = 2; i < RING - 1; i += 2) {
            issue_k();
            if (i + 1 < RING - 1) issue_v();
        }
        // (an even ring has keys under way last, and goes on with their values; an odd one with the next keys)
        auto issue_next = [&](bool behind_keys) {
            if (behind_keys == (RING % 2 == 0)) issue_v();
            else issue_k();
        };
        const float scale = rsqrtf((float)D) * kLog2e;
        A q[KS][2];
        float back = 1.f;           // what scores are multiplied by
        {
            float4 x[KS];
            float high = 0.f, low = INFINITY;
            auto least = [&](float y) { low = y != 0.f ? fminf(low, fabsf(y)) : low; };
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                x[ks] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (head < r.heads) x[ks] = *reinterpret_cast<const float4*>(r.q + head * D + (c + 4 * (ks >> 1)) * 8 + (ks & 1) * 4);
                if (A::kScaled) {
                    high = fmaxf(fmaxf(fmaxf(high, fabsf(x[ks].x)), fmaxf(fabsf(x[ks].y), fabsf(x[ks].z))), fabsf(x[ks].w));
                    least(x[ks].x); least(x[ks].y); least(x[ks].z); least(x[ks].w);
                }
            }
            float by = scale;
            if (A::kScaled) {
                high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 1));
                high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 2));
                // What the largest leaves of the others: 2^-39 of it.  Up to 1024 that is 2^-29, which a key would have to be
                // in the thousands for to be seen; beyond, where there are others that it takes bits from, the range is
                // worked out by fp32 instructions.
                if (__any_sync(0xffffffffu, high > 1024.f && low < high * 0x1p-17f)) {
                    copy_wait<0>();
                    __syncwarp();
                    lost = true;
                    return true;
                }
                // the largest query becomes 2^14 to 2^15
                const int up = min(max(14 - ilogbf(fmaxf(high, 1e-36f)), -110), 110);
                by = ldexpf(1.f, up);
                back = ldexpf(scale, -up);
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                q[ks][0].set(x[ks].x * by, x[ks].y * by);
                q[ks][1].set(x[ks].z * by, x[ks].w * by);
            }
        }
#pragma unroll
        for (int i = 0; i < D / 8; i++) o[i] = make_float2(0.f, 0.f);
        m = -INFINITY;
        l = 0.f;
        int up = 0, steps = 0;
        bool stopped = false;
#pragma unroll 1
        for (int pos = r.begin; pos < r.end; pos += UNIT) {
            if (flag != nullptr && (++steps & 7) == 0) {
                if (__any_sync(0xffffffffu, up)) {
                    stopped = true;
                    break;
                }
                up = ld_flag(flag);
            }
            // ---- scores of keys 8 j + 2 c and 8 j + 2 c + 1 ----
            uint32_t from = ring.take();
            __syncwarp();
            // (sums of 64 dimensions within the tensor core, the rest outside)
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int i = 0; i < D / 32; i += 2) {
                float d[2][4];
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    uint4 k[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) k[j] = read16(from + (8 * j + g) * 2 * D + ((c + 4 * (i + x)) ^ ((g & 1) << 2)) * 16);
#pragma unroll
                    for (int j = 0; j < 2; j++) mma_rows(d[j], q[2 * (i + x)][0], q[2 * (i + x)][1], k[j].x, k[j].y, x == 0);
#pragma unroll
                    for (int j = 0; j < 2; j++) mma_rows(d[j], q[2 * (i + x) + 1][0], q[2 * (i + x) + 1][1], k[j].z, k[j].w, false);
                }
#pragma unroll
                for (int j = 0; j < 2; j++) sum[j] = add2(sum[j], add2(make_float2(d[j][0], d[j][1]), make_float2(d[j][2], d[j][3])));
            }
            issue_next(true);
            const unsigned now = there >> (RING - 1) / 2 * 4;            // (as many steps are ahead of this one)
            float s[4] = {sum[0].x, sum[0].y, sum[1].x, sum[1].y};
            if (A::kHalves) {
#pragma unroll
                for (int u = 0; u < 4; u++) s[u] += __shfl_xor_sync(0xffffffffu, s[u], 16);
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (A::kScaled) s[u] *= back;
                if (!(now >> u & 1)) s[u] = -INFINITY;
                top = fmaxf(top, s[u]);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (__any_sync(0xffffffffu, top != m)) {
                const float by = top == m ? 1.f : exp2_fast(m - top);
                l *= by;
#pragma unroll
                for (int i = 0; i < D / 8; i++) o[i] = make_float2(o[i].x * by, o[i].y * by);
                m = top;
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                s[u] = s[u] == -INFINITY ? 0.f : exp2_fast(s[u] - top + A::kLift);
                l += s[u];
            }
            A p[2];
            p[0].set(s[0], s[1]);
            p[1].set(s[2], s[3]);
            // ---- sums over the values ----
            from = ring.take();
            __syncwarp();
#pragma unroll
            for (int i = 0; i < D / 64; i++) {
                uint32_t w[4][4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const uint4 v = read16(from + (2 * c + (u & 1) + 8 * (u >> 1)) * 2 * D + ((g + 8 * i) ^ 2 * c) * 16);
                    w[u][0] = v.x; w[u][1] = v.y; w[u][2] = v.z; w[u][3] = v.w;
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int sel = j & 1 ? 0x7632 : 0x5410;
                    float d[4];
                    mma_rows(d, p[0], p[1], __byte_perm(w[0][j >> 1], w[1][j >> 1], sel), __byte_perm(w[2][j >> 1], w[3][j >> 1], sel), true);
                    o[8 * i + j] = add2(o[8 * i + j], add2(make_float2(d[0], d[1]), make_float2(d[2], d[3])));
                }
            }
            issue_next(false);
        }
        copy_wait<0>();
        if (stopped) return false;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        float all = l;
#pragma unroll
        for (int i = 0; i < D / 8; i++) {
            if (A::kLift != 0.f) o[i] = make_float2(o[i].x * (1.f / 32768.f), o[i].y * (1.f / 32768.f));
            if (A::kHalves) o[i] = add2(o[i], make_float2(__shfl_xor_sync(0xffffffffu, o[i].x, 16), __shfl_xor_sync(0xffffffffu, o[i].y, 16)));
            all += fabsf(o[i].x) + fabsf(o[i].y);
        }
        if (A::kLift != 0.f) l *= 1.f / 32768.f;
        lost = __any_sync(0xffffffffu, head < r.heads && split_sum_lost(all));
        return true;
    }
    __device__ __forceinline__ void store(const PagedRow& r, float* at, int stride, bool finished) const {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        if (lost) {
            paged_again<C, D>(r, spare, at, stride, finished);
            return;
        }
        if (g >= r.heads) return;
        const float by = !finished ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < D / 64; i++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    *reinterpret_cast<float4*>(at + g * stride + 64 * i + 16 * c + 8 * e + j) =
                        e ? make_float4(o[8 * i + j].y * by, o[8 * i + j + 1].y * by, o[8 * i + j + 2].y * by, o[8 * i + j + 3].y * by)
                          : make_float4(o[8 * i + j].x * by, o[8 * i + j + 1].x * by, o[8 * i + j + 2].x * by, o[8 * i + j + 3].x * by);
        if (!finished && c == 0) *reinterpret_cast<float2*>(at + g * stride + D) = make_float2(m, l);
    }
};

// ---- division of the work -------------------------------------------------------------------------------------------------
// Two forms.  Without parts (wpp > 0): a pass over one row's keys belongs to wpp warps of one block.  With parts (wpp = 0): the keys of
// all rows together, in units of a warp's step, are divided among all warps of the grid in equal consecutive ranges, whatever the
// rows' lengths; a pass that several blocks share leaves a part per block, which reef_paged_attention_join brings together in the
// order of the keys: no block waits for another and nothing depends on which one comes first.
constexpr int kPagedSlotsOfBlock = 2 + 8;   // parts of a block, first ranges of its warps
constexpr int kPagedMinUnits = 2;        // units of a warp at least, before further warps take part
struct PagedSlots {
    int pair[16];                        // pass of a warp's first and last, unfinished range; -1: none
    int ends[16];                        // 1: the range begins the pass, 2: it ends it
    int token[8];                        // the token that a warp begins with
    int before[8];                       // units of the tokens before that one, of one pass each
    int sums[8];
};
template <class E>
__device__ __forceinline__ bool paged_attention_body(const KTask& t, int vb, unsigned char* smem, const int* flag) {
    const PagedP& p = t.p.paged;
    const int4* tok = (const int4*)t.a[4];
    float* out = (float*)t.a[5];
    PagedSlots& sl = *reinterpret_cast<PagedSlots*>(smem);
    // A warp's slots: its last range goes over the engine's scratch memory; its first, when others follow, behind the block's parts.
    constexpr int stride = paged_stride(E::DIM), slot_floats = E::GB * stride;
    static_assert(slot_floats * 4 <= E::SCRATCH && sizeof(PagedSlots) + 16 + 8 * E::SCRATCH <= 227 * 1024, "shared memory");
    char* const scratch = reinterpret_cast<char*>(smem) + ((sizeof(PagedSlots) + 15) & ~15);
    float* const parts = p.wpp > 0 ? nullptr : (float*)t.a[6] + 2 * ((t.nblocks + 1) & ~1) + (size_t)vb * kPagedSlotsOfBlock * slot_floats;
    auto slot = [&](int s) { return s & 1 ? reinterpret_cast<float*>(scratch + (s >> 1) * E::SCRATCH) : parts + (2 + (s >> 1)) * slot_floats; };
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
    auto range = [&](int token, int x, int4 tk, int a, int b, int n, int s) {
        const int kh = x / p.subs, h0 = kh * group + (x - kh * p.subs) * E::GB;
        const PagedRow r = {(const float*)t.a[0] + (size_t)token * p.qs + p.qo + (size_t)h0 * E::DIM, (const char*)t.a[1], (const char*)t.a[2],
                            (const int*)t.a[3] + (size_t)tk.y * p.mp, min(E::GB, (kh + 1) * group - h0), a * E::UNIT,
                            min(b * E::UNIT, paged_length(p, tk)), p.ps, p.pages, p.kvh, kh, p.ps_mul, p.ps_shift};
        if (!e.run(r, scratch + warp * E::SCRATCH, flag)) return false;
        if (a == 0 && b == n) {
            e.store(r, out + ((size_t)token * p.heads + h0) * E::DIM, E::DIM, true);
        } else {
            __syncwarp();
            e.store(r, slot(s), stride, false);
            if (lane == 0) {
                sl.pair[s] = token * P + x;
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
            if (a < b) stopped = !range(token, (int)(pair - (long long)token * P), tk, a, b, n, 2 * warp + 1);
            if (n == 0 && i == 0) {
                int heads;
                float* at = where_out((int)pair, &heads);
                for (int c = lane * 4; c < heads * E::DIM; c += 128) *reinterpret_cast<float4*>(at + c) = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    } else {
        // units of the tokens before each (fewer than 2^31 in all: the plan sees to it); up to 32 tokens every warp counts for itself
        auto units_of = [&](int i) { return (paged_length(p, tok[i]) + E::UNIT - 1) / E::UNIT; };
        auto scan = [&](int v) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            return v;
        };
        int all = 0, upto, mine = 0, u, end, token = 0, base = 0;
        // block vb's units of all, and within them warp w's
        int lo = 0, len = 0;
        auto divide = [&]() {
            const int W = all * P, blocks = min(t.nblocks, (W + 8 * kPagedMinUnits - 1) / (8 * kPagedMinUnits));
            const int each = blocks > 0 ? W / blocks : 0, more = W - each * blocks;
            lo = vb < blocks ? vb * each + min(vb, more) : 0;
            len = vb < blocks ? each + (vb < more ? 1 : 0) : 0;
        };
        auto begin_of = [&](int w) { return lo + (int)((unsigned)len * w >> 3); };
        if (p.tokens <= 32) {
            mine = lane < p.tokens ? units_of(lane) : 0;
            upto = scan(mine);
            all = __shfl_sync(0xffffffffu, upto, 31);
            divide();
            u = begin_of(warp);
            end = begin_of(warp + 1);
            token = __popc(__ballot_sync(0xffffffffu, upto * P <= u));
            base = __shfl_sync(0xffffffffu, (upto - mine) * P, token & 31);
            __syncthreads();             // (the slots are empty)
        } else {
            // a run of tokens to a thread
            const int per = (p.tokens + kThreads - 1) / kThreads, t0 = min(p.tokens, tid * per), t1 = min(p.tokens, t0 + per);
            for (int i = t0; i < t1; i++) mine += units_of(i);
            upto = scan(mine);
            if (lane == 31) sl.sums[warp] = upto;
            __syncthreads();
            int before = 0;
#pragma unroll
            for (int w = 0; w < 8; w++) {
                if (w < warp) before += sl.sums[w];
                all += sl.sums[w];
            }
            upto += before;
            divide();
            if (mine > 0 && (upto - mine) * P < lo + len && upto * P > lo)
                for (int w = 0; w < 8; w++) {
                    const int at = begin_of(w);
                    if (at < (upto - mine) * P || at >= upto * P) continue;
                    int b = upto - mine, i = t0;
                    for (; i < t1; i++) {
                        const int n = units_of(i);
                        if (at < (b + n) * P) break;
                        b += n;
                    }
                    sl.token[w] = i;
                    sl.before[w] = b;
                }
            __syncthreads();
            u = begin_of(warp);
            end = begin_of(warp + 1);
            if (u < end) {
                token = sl.token[warp];
                base = sl.before[warp] * P;
            }
        }
        if (u < end) {
            while (u < end && token < p.tokens) {
                const int4 tk = tok[token];
                const int n = (paged_length(p, tk) + E::UNIT - 1) / E::UNIT;
                if (u >= base + n * P) {
                    base += n * P;
                    token++;
                    continue;
                }
                const int r = (u - base) / n, a = u - base - r * n, b = min(n, a + (end - u));
                if (!range(token, r, tk, a, b, n, 2 * warp + (u + (b - a) == end ? 1 : 0))) {
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
    // ranges of one pass lie side by side: the lane of the first of them says which they are, all threads bring their values together
    const int pair = lane < 16 ? sl.pair[lane] : -1, ends = lane < 16 ? sl.ends[lane] : 0;
    const unsigned used = __ballot_sync(0xffffffffu, pair >= 0), chain = __match_any_sync(0xffffffffu, pair) & used;
    const int last = 31 - __clz(chain | 1);
    const int both = (ends & 1) | (__shfl_sync(0xffffffffu, ends, last) & 2);
    unsigned heads_of = __ballot_sync(0xffffffffu, pair >= 0 && (chain & ((1u << lane) - 1)) == 0);
    int left[2] = {-1, -1};             // what this block leaves: a pass that began earlier, one that goes on behind it
    while (heads_of) {
        const int s = __ffs(heads_of) - 1;
        heads_of &= heads_of - 1;
        const int id = __shfl_sync(0xffffffffu, pair, s), e = __shfl_sync(0xffffffffu, both, s);
        const unsigned slots = __shfl_sync(0xffffffffu, chain, s);
        int heads;
        float* at = where_out(id, &heads);
        int step = E::DIM;
        if (e != 3) {
            at = parts + (e & 1) * slot_floats;     // (only with parts)
            step = stride;
            left[e & 1] = id;
        }
        for (int i = tid; i < heads * (E::DIM / 4); i += kThreads) {
            const int j = i / (E::DIM / 4), c = (i - j * (E::DIM / 4)) * 4;
            float top = -INFINITY, sum = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < 16; x++)
                if (slots >> x & 1) top = fmaxf(top, slot(x)[j * stride + E::DIM]);
#pragma unroll
            for (int x = 0; x < 16; x++) {
                if (!(slots >> x & 1)) continue;
                const float* from = slot(x) + j * stride;
                const float2 ml = *reinterpret_cast<const float2*>(from + E::DIM);
                const float4 y = *reinterpret_cast<const float4*>(from + c);
                const float by = ml.x == top ? 1.f : exp2_fast(ml.x - top);
                sum = fmaf(ml.y, by, sum);
                o.x = fmaf(y.x, by, o.x); o.y = fmaf(y.y, by, o.y); o.z = fmaf(y.z, by, o.z); o.w = fmaf(y.w, by, o.w);
            }
            const float by = e != 3 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<float4*>(at + (size_t)j * step + c) = make_float4(o.x * by, o.y * by, o.z * by, o.w * by);
            if (e != 3 && c == 0) *reinterpret_cast<float2*>(at + (size_t)j * step + E::DIM) = make_float2(top, sum);
        }
    }
    if (p.wpp == 0 && tid == 0) {
        int* desc = (int*)t.a[6] + 2 * vb;
        desc[0] = left[0];
        desc[1] = left[1];
    }
    return true;
}

// ---- shapes ---------------------------------------------------------------------------------------------------------------
constexpr int kSmsPlanned = 148;                           // launch geometry is planned without a GPU
// Tensor cores from three query heads to a 16-bit key head on.
__host__ inline int paged_heads_of_a_pass(int kt, int d, int group) {
    if (kt != KT_FP32) return group <= 2 ? group : group <= 4 ? 4 : 8;
    const int most = d == 256 ? 4 : 8, passes = (group + most - 1) / most, gb = (group + passes - 1) / passes;
    return gb == 7 ? 8 : gb;
}
__host__ inline bool paged_mma(const PagedP& p) { return p.kt != KT_FP32 && p.gb > 2; }
struct PagedSimtShape { int unit, scratch; };
__host__ inline PagedSimtShape paged_simt_shape(const PagedP& p) {      // UNIT and SCRATCH of PagedSimt
    const int vec = p.kt == KT_FP32 ? 4 : 8, lanes = p.d / vec > 32 ? 32 : p.d / vec, pieces = p.d / (vec * lanes), keys = paged_simt_keys(pieces, lanes, p.gb);
    const int ring = kPagedSimtRing * keys * pieces * 512, slot = p.gb * paged_stride(p.d) * 4;
    return {32 / lanes * keys, ring > slot ? ring : slot};
}
__host__ inline int paged_unit(const PagedP& p) { return paged_mma(p) ? 16 : paged_simt_shape(p).unit; }      // keys of a warp's step
__host__ inline int paged_attention_smem(const PagedP& p) {
    return (int)((sizeof(PagedSlots) + 15) & ~15) + 8 * (paged_mma(p) ? paged_mma_scratch(p.d, p.gb) : paged_simt_shape(p).scratch);
}
__host__ inline int paged_blocks_per_sm(const PagedP& p) { return paged_mma(p) ? 1 : 2; }
// Warps of a pass where no parts are left: a second, fourth or eighth shortens a pass, and costs a join and, where there are passes enough for
// all warps, further rounds of blocks.  Measured in 1, 2, 4 and 8 warps (us): fp32 instructions, 1536 passes of up to 32 units 26.8, 29.1, 28.2,
// 32.9, of 128 units 94, 80, 73, 68; 384 of 32 units 20.6, 16.6, 12.4, 12.4; 1832 of 16 units 22, 27, 28, 37.  Tensor cores, 2048 passes of 8 units
// 22.7, 36.9, 45.1, 65.6; 32 units 66, 72, 80, 102; 128 units 228, 201, 191, 201; 512 passes of 32 units 36.9, 24.7, 24.7, 28.8.  So as many as it
// takes to have warps for two thirds of the machine, or no more than 16 units a warp, 32 on the tensor cores.
__host__ inline int paged_warps_of_a_pass(const PagedP& p, long long passes, int units) {
    const int blocks = paged_blocks_per_sm(p), most = 32 / blocks;
    int w = 1;
    while (w < 8 && w < units && (passes * w < 768 * blocks || units > most * w)) w *= 2;
    return w;
}
// Blocks of the form with parts: what the SMs hold at once, fewer where the longest rows would not give every warp its least work.  (SMs do
// not get the same share of the memory's bandwidth: of 148 equal shares of 860 MB one was through after 102 us and one after 145.  Two or
// three times as many blocks, to be taken by whichever SM is free, brought 157 to 152 us with two blocks to an SM, and cost more in
// further parts and their join.)
__host__ inline int paged_parts_blocks(const PagedP& p, long long units) {
    const long long want = (units + 8 * kPagedMinUnits - 1) / (8 * kPagedMinUnits), slots = (long long)paged_blocks_per_sm(p) * kSmsPlanned;
    return (int)(want < slots ? want : slots);
}
__host__ inline size_t paged_parts_bytes(const PagedP& p, int blocks) {
    return ((size_t)2 * ((blocks + 1) & ~1) + (size_t)blocks * kPagedSlotsOfBlock * p.gb * paged_stride(p.d)) * 4;
}

// ---- join -----------------------------------------------------------------------------------------------------------------
// args: parts, out.  A pass that block b left unfinished: its part, then those of the blocks behind it that lie in the same pass, added in
// their order.  Few parts: a warp to a head of a pass.  Many (a long row): a block to 32 dimensions of a head, the parts divided
// among groups of eight lanes, the groups added in their order.
constexpr int kJoinFew = 16;
__host__ __device__ inline int paged_join_blocks(int blocks, int gb) { return min((blocks * gb + 7) / 8, 2 * kSmsPlanned); }
__device__ __forceinline__ bool body_paged_join(const KTask& t, int vb, unsigned char* smem, const int*) {
    const PagedP& p = t.p.paged;
    const int blocks = p.split, gb = p.gb, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = p.d;
    const int stride = paged_stride(D), P = p.kvh * p.subs, group = p.heads / p.kvh;
    const int* desc = (const int*)t.a[0];
    const float* parts = (const float*)t.a[0] + 2 * ((blocks + 1) & ~1);
    float* out = (float*)t.a[1];
    int2* left = reinterpret_cast<int2*>(smem);                   // a copy of the blocks' words
    int* many = reinterpret_cast<int*>(left + blocks);            // blocks that begin a pass of many parts
    float* red = reinterpret_cast<float*>(smem + (blocks * 12 + 15) / 16 * 16);   // 32 groups x 36
    __shared__ int n_many;
    __syncthreads();                           // a persistent caller's previous block is out of shared memory
    for (int b = tid; b < blocks; b += kThreads) left[b] = reinterpret_cast<const int2*>(desc)[b];
    if (tid == 0) n_many = 0;
    __syncthreads();
    auto count = [&](int b) {                  // parts of the pass that block b begins
        const int id = left[b].y;
        int n = 1;
        for (;; n += 32) {
            const unsigned more = __ballot_sync(0xffffffffu, b + n + lane < blocks && left[min(b + n + lane, blocks - 1)].x == id);
            if (more != 0xffffffffu) return n + __ffs(~more) - 1;
        }
    };
    auto is_long = [&](int b) { return left[b].y >= 0 && b + kJoinFew < blocks && left[b + kJoinFew].x == left[b].y; };
    auto at = [&](int b, int j, int i) { return parts + ((size_t)(b + i) * kPagedSlotsOfBlock + (i == 0 ? 1 : 0)) * gb * stride + j * stride; };
    // the place of a head in `out`, -1 for a head that is none
    auto place = [&](int id, int j) {
        if (id < 0 || id >= p.tokens * P) return -1LL;
        const int token = id / P, r = id - token * P, kh = r / p.subs, h = kh * group + (r - kh * p.subs) * gb + j;
        return h < (kh + 1) * group ? ((long long)token * p.heads + h) * D : -1LL;
    };
    const int grid = t.nblocks;
    for (int item = vb * 8 + warp; item < blocks * gb; item += grid * 8) {
        const int b = item / gb, j = item - b * gb;
        const long long to = place(left[b].y, j);
        if (to < 0) continue;
        if (is_long(b)) continue;
        const int n = min(count(b), kJoinFew);
        const float mine = lane < n ? at(b, j, lane)[D] : -INFINITY;
        const float top = warp_max(mine), by = mine == top ? 1.f : exp2_fast(mine - top);
        float sum = 0.f;
        float4 o[2];
        o[0] = o[1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < n; i++) {
            const float* x = at(b, j, i);
            const float f = __shfl_sync(0xffffffffu, by, i);
            sum = fmaf(x[D + 1], f, sum);
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (k * 128 + lane * 4 < D) {
                    const float4 y = *reinterpret_cast<const float4*>(x + k * 128 + lane * 4);
                    o[k].x = fmaf(y.x, f, o[k].x); o[k].y = fmaf(y.y, f, o[k].y); o[k].z = fmaf(y.z, f, o[k].z); o[k].w = fmaf(y.w, f, o[k].w);
                }
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (k * 128 + lane * 4 < D)
                *reinterpret_cast<float4*>(out + to + k * 128 + lane * 4) = make_float4(o[k].x * inv, o[k].y * inv, o[k].z * inv, o[k].w * inv);
    }
    // (which come first does not matter: each is a result of its own)
    for (int b = tid; b < blocks; b += kThreads)
        if (is_long(b)) many[atomicAdd(&n_many, 1)] = b;
    __syncthreads();
    const int slices = D / 32, g = tid >> 3, c = (tid & 7) * 4;
    for (int item = vb; item < n_many * gb * slices; item += grid) {
        // in the order of the blocks, which is the same in every block of this grid
        const int k = item / (gb * slices), j = (item - k * gb * slices) / slices, d0 = (item % slices) * 32;
        int b = -1;
        for (int i = 0; i < n_many; i++) {
            int rank = 0;
            for (int o = 0; o < n_many; o++) rank += many[o] < many[i];
            if (rank == k) b = many[i];
        }
        const long long to = place(left[b].y, j);
        if (to < 0) continue;                  // (the same for all threads)
        const int n = count(b);
        float top = -INFINITY;
        for (int i = lane; i < n; i += 32) top = fmaxf(top, at(b, j, i)[D]);
        top = warp_max(top);                   // (every warp for itself)
        float sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = g; i < n; i += 32) {
            const float* x = at(b, j, i);
            const float2 ml = *reinterpret_cast<const float2*>(x + D);
            const float4 y = *reinterpret_cast<const float4*>(x + d0 + c);
            const float by = ml.x == top ? 1.f : exp2_fast(ml.x - top);
            sum = fmaf(ml.y, by, sum);
            o.x = fmaf(y.x, by, o.x); o.y = fmaf(y.y, by, o.y); o.z = fmaf(y.z, by, o.z); o.w = fmaf(y.w, by, o.w);
        }
        __syncthreads();                       // the item before is out of `red`
        *reinterpret_cast<float4*>(red + g * 36 + c) = o;
        if (c == 0) red[g * 36 + 32] = sum;
        __syncthreads();
        if (tid < 32) {
            float total = 0.f, v = 0.f;
#pragma unroll 8
            for (int i = 0; i < 32; i++) {
                v += red[i * 36 + tid];
                total += red[i * 36 + 32];
            }
            out[to + d0 + tid] = total == 0.f ? 0.f : v / total;
        }
    }
    return true;
}
__host__ inline int paged_join_smem(int blocks) { return (blocks * 12 + 15) / 16 * 16 + 32 * 36 * 4; }

}  // namespace reef
