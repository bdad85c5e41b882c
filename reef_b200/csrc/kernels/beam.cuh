// Beam search's selection: of every request the `beams` best continuations over its beams and the vocabulary,
//   cand(b, w) = score[b] + logits[b][w] - log sum_u exp(logits[b][u]),
// ties by the lower beam, then the greater logit, then the lower word.  A beam that has ended (live 0) competes with its score and the end word alone; candidates of
// -infinity or NaN are none, so a row without a finite sum (a NaN, an infinity, nothing but -infinity) has none, nor has a beam without a
// finite score.  What is missing comes out as token -1, parent -1, score -infinity, live 0.
#pragma once
#include "paged_cache.cuh"

namespace reef {

constexpr int kBeamMax = 16;
constexpr int kBeamVecs = 4;                              // 128-bit loads of a lane and turn
constexpr int kBeamTurn = kBeamVecs * 4 * 32;             // words of a warp's turn
constexpr int kBeamRoom = 512;                            // candidates that a block ranks side by side
// Parts of a row of logits, a part to a block: a turn of its eight warps at least, and over all rows not more than four blocks to an SM
// (a second round of blocks repeats what a block has to do once: 256 rows in 2 parts each 23 us, in 4 parts 27, in 1 part 31).
__host__ inline int beam_parts(long long rows, int vocab) {
    const long long least = 8LL * kBeamTurn, most = (vocab + least - 1) / least, slots = 4 * 148;
    if (rows * most <= slots) return (int)most;
    if (rows <= slots) return (int)(slots / rows);
    return 1;
}
__host__ __device__ inline int beam_part_floats(int beams) { return 2 + 2 * beams; }

// V: values, I: what decides between equal ones, the lowest first
template <class V, class I>
struct BeamRoom {
    V value[kBeamRoom];
    I index[kBeamRoom];
    V line[8];
    I who[8];
    int count;
};
typedef unsigned long long BeamKey;
constexpr int kBeamSmem = (int)sizeof(BeamRoom<double, BeamKey>);

template <class V, class I>
__device__ __forceinline__ bool beam_before(V a, I ia, V b, I ib) { return a > b || (a == b && ia < ib); }

// `each(f)` calls f(value, index) for the values of this thread; -infinity and NaN are none.  block_collect gathers those of all threads (s.count
// is 0 before, the threads have not met behind it), block_place ranks them, if there is room for all, ties by the lowest index, and calls
// `take(i, value, index)` for the i-th of the K greatest; both it and block_top return how many of these there are.
template <class V, class I, class Each>
__device__ __forceinline__ void block_collect(BeamRoom<V, I>& s, Each each) {
    each([&](V v, I i) {
        if (v > (V)-INFINITY) {
            const int at = atomicAdd(&s.count, 1);
            if (at < kBeamRoom) {
                s.value[at] = v;
                s.index[at] = i;
            }
        }
    });
}
template <class V, class I, class Take>
__device__ __forceinline__ int block_place(int K, const BeamRoom<V, I>& s, int n, Take take) {
    for (int c = threadIdx.x; c < n; c += kThreads) {
        const V v = s.value[c];
        const I i = s.index[c];
        int r = 0;
#pragma unroll 4
        for (int o = 0; o < n; o++) r += beam_before(s.value[o], s.index[o], v, i);
        if (r < K) take(r, v, i);
    }
    return min(n, K);
}
// Every warp's K-th greatest of its lanes' values has K values at or above it, so the greatest of these eight is a line that few values reach.
// (s.count is 0 behind it.)
template <class V, class I>
__device__ __forceinline__ V block_line(int K, BeamRoom<V, I>& s, V top) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < 32; j++) {
        const V v = __shfl_sync(0xffffffffu, top, j);
        rank += v > top || (v == top && j < lane);
    }
    __syncthreads();
    if (rank == K - 1) s.line[warp] = top;
    if (tid == 0) s.count = 0;
    __syncthreads();
    V line = s.line[0];
#pragma unroll
    for (int w = 1; w < 8; w++) line = s.line[w] > line ? s.line[w] : line;
    return line;
}
// The line is drawn through the threads' maxima.  Where more reach it than there is room for (many equal values) the best one behind the last is looked for K times.
template <class V, class I, class Each, class Take>
__device__ __forceinline__ int block_top(int K, BeamRoom<V, I>& s, Each each, Take take) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const V ninf = -INFINITY;
    V top = ninf;
    each([&](V v, I) { if (v > top) top = v; });
    const V line = block_line(K, s, top);
    block_collect(s, [&](auto f) { each([&](V v, I i) { if (v >= line) f(v, i); }); });
    __syncthreads();
    const int n = s.count;
    if (n <= kBeamRoom) return block_place(K, s, n, take);
    constexpr I none = sizeof(I) == 4 ? (I)0x7fffffff : ~(I)0;
    V last = INFINITY;
    I last_i = (I)-1;               // (of the keys it is the highest, but their values are finite)
    int found = 0;
    for (; found < K; found++) {
        V best = ninf;
        I best_i = none;
        each([&](V v, I i) {
            if (v > ninf && beam_before(last, last_i, v, i) && beam_before(v, i, best, best_i)) best = v, best_i = i;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const V v = __shfl_xor_sync(0xffffffffu, best, o);
            const I i = __shfl_xor_sync(0xffffffffu, best_i, o);
            if (beam_before(v, i, best, best_i)) best = v, best_i = i;
        }
        __syncthreads();
        if (lane == 0) s.line[warp] = best, s.who[warp] = best_i;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++)
            if (beam_before(s.line[w], s.who[w], best, best_i)) best = s.line[w], best_i = s.who[w];
        if (best == ninf) break;
        if (tid == 0) take(found, best, best_i);
        last = best;
        last_i = best_i;
    }
    return found;
}

// row of logits of a beam; -1: it has none
__device__ __forceinline__ int beam_logits(const BeamP& p, const int* start, int r) {
    if (start == nullptr) return r;
    const int a = start[r], b = start[r + 1];
    return b > a && b > 0 && b <= p.tokens ? b - 1 : -1;
}

// ---- scan: a part of a row of logits -> its maximum, the sum of exponentials below it, its `beams` greatest ------------------
// args: logits, live, [start], parts.  One pass, a range of the part to a warp, no warp waiting for another until the end: a lane carries the
// maximum of its words, the turn that it came in, and a sum below it; the next turn's loads are under way while a turn is looked at.  The lanes
// are divided into 16 groups, or 32 for more beams than 8, whose words lie all over the part.  K groups have a word at or above the K-th
// greatest of their maxima, so nothing but what reaches that line (words above it, and those equal to it up to its turn) can be among
// the K greatest.  The words of the lanes whose maxima reach it, some 12 of 256, are read again, from L2, and those that do are ranked.
// 256 rows of 100003 words, 102 MB, 26 us from HBM (0.60 of the measured copy rate), 23 with most of it in L2 (39 with the greatest words kept in
// order as they came, 61 with a room in shared memory that was ranked whenever it filled); 22 and 19 of these are the pass, the rest the
// line, the second look and the ranking, during which little is read; four rows of 30522 words 6.  Code of many unrolled steps after the pass is itself slow, every line of
// it being fetched once: a loop unrolled 16 times took 1 us longer than the loop.
struct BeamScan {
    BeamRoom<float, int> room;
    float key[8][32];            // of every warp and group the greatest word and the turn it came in
    int turn[8][32];
    float top[8], sum[8];
};
__device__ __forceinline__ float2 exp_two(float x, float y, float top) {     // e^(x - top), e^(y - top)
    float2 d = add2(make_float2(x, y), make_float2(-top, -top));
    d = fma2(d, make_float2(kLog2e, kLog2e), make_float2(0.f, 0.f));
    return make_float2(exp2_fast(d.x), exp2_fast(d.y));
}
__device__ __forceinline__ bool body_beam_scan(const KTask& t, int vb, unsigned char* smem, const int* flag) {
    const BeamP& p = t.p.beam;
    const int r = vb / p.parts, part = vb - r * p.parts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.beams;
    const int* live = (const int*)t.a[1];
    const int* start = p.has_start ? (const int*)t.a[2] : nullptr;
    float* out = (float*)t.a[2 + p.has_start] + (size_t)vb * beam_part_floats(K);
    if (live[r] == 0) return true;
    const int row = beam_logits(p, start, r);
    if (row < 0) return true;
    BeamScan& s = *reinterpret_cast<BeamScan*>(smem);
    // loads begin at a 16-byte boundary: up to three words of the row before are masked
    const float* logits = (const float*)t.a[0] + (size_t)row * p.vocab;
    const int lead = (int)(((size_t)row * p.vocab) & 3);
    const int first = part * p.part, loads = min(p.part, (p.vocab + lead + 3) / 4 - first);         // 128-bit loads of this part
    const int each_warp = loads > 0 ? ((loads + 7) / 8 + 31) / 32 * 32 : 0;
    const int begin = (first + warp * each_warp) * 4 - lead, end = min(p.vocab, (first + min(loads, (warp + 1) * each_warp)) * 4 - lead);
    float4 x[kBeamVecs], next[kBeamVecs];
    auto load_at = [&](int w, int end) {
        if (w >= 0 && w + 4 <= end) return *reinterpret_cast<const float4*>(logits + w);
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; e++) z[e] = w + e >= 0 && w + e < end ? logits[w + e] : -INFINITY;
        return make_float4(z[0], z[1], z[2], z[3]);
    };
    auto load = [&](float4 (&y)[kBeamVecs], int at) {
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++) y[i] = load_at(at + (i * 32 + lane) * 4, end);
    };
    int here = begin, turn = 0;                // first word of this turn, and of the one with this lane's maximum
    float top = -INFINITY;
    float2 sum = make_float2(0.f, 0.f);
    bool stopped = false;
    int up = 0, turns = 0;
    load(x, begin);
#pragma unroll 1
    for (; here < end; here += kBeamTurn) {
        if (flag != nullptr && (++turns & 3) == 0) {       // best-effort flavour: a look at the preempt flag, asked for ahead
            if (__any_sync(0xffffffffu, up)) {
                stopped = true;
                break;
            }
            up = ld_flag(flag);
        }
        if (here + kBeamTurn < end) load(next, here + kBeamTurn);
        float high = -INFINITY;
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++) high = fmaxf(high, fmaxf(fmaxf(x[i].x, x[i].y), fmaxf(x[i].z, x[i].w)));
        if (high > top) {
            const float by = exp2_fast((top - high) * kLog2e);
            sum.x *= by;
            sum.y *= by;
            top = high;
            turn = here;
        }
        if (top == -INFINITY) {
#pragma unroll
            for (int i = 0; i < kBeamVecs; i++) {       // (a NaN is not lost)
                const float v = x[i].x + x[i].y + x[i].z + x[i].w;
                if (v != v) sum.x += v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kBeamVecs; i++) {
                const float2 a = exp_two(x[i].x, x[i].y, top), b = exp_two(x[i].z, x[i].w, top);
                sum = add2(sum, add2(a, b));
            }
        }
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++) x[i] = next[i];
    }
    // the warps' sums and their groups' maxima meet
    const float high = warp_max(top), part_sum = sum.x + sum.y;
    const float total = warp_sum(top == -INFINITY ? part_sum : part_sum * exp2_fast((top - high) * kLog2e));
    const int groups = K <= 8 ? 16 : 32;
    float key = top;
    int key_turn = turn;
    if (groups == 16) {
        const float v = __shfl_xor_sync(0xffffffffu, key, 16);
        const int i = __shfl_xor_sync(0xffffffffu, key_turn, 16);
        if (beam_before(v, i, key, key_turn)) key = v, key_turn = i;
    }
    __syncthreads();                           // a persistent caller's previous block is out of shared memory
    if (lane == 0) {
        s.top[warp] = high;
        s.sum[warp] = total;
    }
    if (lane < groups) {
        s.key[warp][lane] = key;
        s.turn[warp][lane] = key_turn;
    }
    if (tid == 0) s.room.count = 0;
    if (__syncthreads_or(stopped)) return false;
    if (warp == 0) {
        const float most_of = lane < 8 ? s.top[lane] : -INFINITY, most = warp_max(most_of);
        const float all = warp_sum(lane >= 8 ? 0.f : most_of == -INFINITY ? s.sum[lane] : s.sum[lane] * exp2_fast((most_of - most) * kLog2e));
        if (lane == 0) {
            out[0] = most;
            out[1] = all;
        }
    }
    // the line, by every warp for itself: a group to a lane
    const int group = lane & (groups - 1);
    key = s.key[0][group];
    key_turn = s.turn[0][group];
#pragma unroll
    for (int w = 1; w < 8; w++) {
        const float v = s.key[w][group];
        const int i = s.turn[w][group];
        if (beam_before(v, i, key, key_turn)) key = v, key_turn = i;
    }
    int rank = 0;
#pragma unroll 2
    for (int j = 0; j < groups; j++) {
        const float v = __shfl_sync(0xffffffffu, key, j);
        const int i = __shfl_sync(0xffffffffu, key_turn, j);
        rank += beam_before(v, i, key, key_turn) || (v == key && i == key_turn && j < group);
    }
    const int at = __ffs(__ballot_sync(0xffffffffu, rank == K - 1)) - 1;
    const float line = __shfl_sync(0xffffffffu, key, at);
    const int line_turn = __shfl_sync(0xffffffffu, key_turn, at), upto = line == -INFINITY ? -0x7fffffff : line_turn + kBeamTurn;
    const unsigned reach = __ballot_sync(0xffffffffu, top > line || (top == line && turn < upto));
    auto each = [&](auto f) {                  // eight lanes to one that reaches the line
        for (unsigned m = reach; m;) {
            unsigned of = m;
            for (int j = lane >> 3; j > 0; j--) of &= of - 1;
            for (int j = 0; j < 4; j++) m &= m - 1;
            if (of == 0) continue;
#pragma unroll 1
            for (int w = begin + (__ffs(of) - 1 + (lane & 7) * 32) * 4; w < end; w += 8 * 8 * 32 * 4) {
                float4 y[8];
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = load_at(w + i * 8 * 32 * 4, end);
                unsigned some = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) some |= (fmaxf(fmaxf(y[i].x, y[i].y), fmaxf(y[i].z, y[i].w)) >= line) << i;
                for (; some; some &= some - 1) {       // (few: a short loop over what is in L1 costs less than the code for all eight)
                    const int at = w + (__ffs(some) - 1) * 8 * 32 * 4;
                    const float4 z = load_at(at, end);
                    const float v[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (v[e] > line || (v[e] == line && at + e < upto)) f(v[e], at + e);
                }
            }
        }
    };
    auto take = [&](int i, float v, int w) {
        out[2 + i] = v;
        out[2 + K + i] = __int_as_float(w);
    };
    block_collect(s.room, each);
    __syncthreads();
    const int n = s.room.count;
    const int found = n <= kBeamRoom ? block_place(K, s.room, n, take) : block_top(K, s.room, each, take);
    if (tid >= found && tid < K) {
        out[2 + tid] = -INFINITY;
        out[2 + K + tid] = __int_as_float(0);
    }
    return true;
}

// ---- pick: the parts of a request's beams -> its new beams --------------------------------------------------------------------
// args: parts, score, live, [start], token, parent, score', live'.  Beams are compared in 64 bits: a score of -50 in 32 bits cannot tell logits
// apart that differ by less than 4e-6.  Where these are equal the lower beam comes first, and within a beam the logits decide, exactly as they
// are (beside a score of -1e30 all of a beam's candidates are equal in 64 bits too), then the lower word: a key of 4, 32 and 28 bits.  Latency: 32 requests of eight beams
// 6 us, one of sixteen beams in 25 parts each 14 (141 when every entry was looked at: the lists are in order, and a line through threads that have
// entries of every rank is a low one).
constexpr int kBeamLists = 4 * 148 + kBeamMax;            // lists of a request at most: parts of all rows, or one of each
__host__ inline int beam_pick_smem() { return kBeamSmem + kBeamMax * (8 + 8 + 4 + 4) + kBeamLists * (8 + 4) + 8; }
__device__ __forceinline__ bool body_beam_pick(const KTask& t, int vb, unsigned char* smem, const int*) {
    const BeamP& p = t.p.beam;
    const int K = p.beams, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, F = beam_part_floats(K);
    const float* parts = (const float*)t.a[0] + (size_t)vb * K * p.parts * F;
    const float* score = (const float*)t.a[1] + (size_t)vb * K;
    const int* live = (const int*)t.a[2];
    const int* start = p.has_start ? (const int*)t.a[3] : nullptr;
    void* const* a = t.a + 3 + p.has_start;
    int* token = (int*)a[0] + (size_t)vb * K;
    int* parent = (int*)a[1] + (size_t)vb * K;
    float* score_out = (float*)a[2] + (size_t)vb * K;
    int* live_out = (int*)a[3] + (size_t)vb * K;
    BeamRoom<double, BeamKey>& s = *reinterpret_cast<BeamRoom<double, BeamKey>*>(smem);
    // of a beam: its logits' maximum, the logarithm of the sum of exponentials below it, its score.  Applied one after the other: their sum
    // would lose the smaller ones where the logits are at the type's lowest value.
    double* log_sum = reinterpret_cast<double*>(smem + kBeamSmem);
    double* base = log_sum + kBeamMax;
    float* highest = reinterpret_cast<float*>(base + kBeamMax);
    int* kind = reinterpret_cast<int*>(highest + kBeamMax);           // 0: no candidates, 1: its parts, 2: it has ended
    double* heads = reinterpret_cast<double*>(kind + kBeamMax);       // the lists' first entries
    int* which = reinterpret_cast<int*>(heads + kBeamLists);          // lists that reach the line
    int* walked = which + kBeamLists;                                 // how many
    __syncthreads();
    for (int b = warp; b < K; b += 8) {
        const int r = vb * K + b;
        int what = 0;
        double norm = 0.0;
        float top = -INFINITY;
        if (live[r] == 0) {
            what = isfinite(score[b]) ? 2 : 0;
        } else if (beam_logits(p, start, r) >= 0) {
            for (int i = lane; i < p.parts; i += 32) top = fmaxf(top, parts[((size_t)b * p.parts + i) * F]);
            top = warp_max(top);
            double sum = 0.0;
            for (int i = lane; i < p.parts; i += 32) {
                const float* x = parts + ((size_t)b * p.parts + i) * F;
                sum += x[0] == -INFINITY && x[1] == 0.f ? 0.0 : (double)x[1] * exp((double)x[0] - top);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            norm = log(sum);
            what = isfinite(norm) && isfinite(top) && isfinite(score[b]) ? 1 : 0;
        }
        if (lane == 0) {
            log_sum[b] = norm;
            base[b] = score[b];
            highest[b] = top;
            kind[b] = what;
        }
    }
    __syncthreads();
    // a list's i-th entry: the value, -infinity for none, and its key
    const int lists = K * p.parts;
    auto key_of = [](int b, unsigned order, int w) { return (BeamKey)b << 60 | (BeamKey)order << 28 | (unsigned)w; };
    auto entry = [&](int list, int i, BeamKey* at) -> double {
        const int b = list / p.parts;
        const float* x = parts + (size_t)list * F + 2 + i;
        const float v = x[0];
        const unsigned bits = __float_as_uint(v + 0.f);          // (-0 as 0), ascending as the logits descend:
        *at = key_of(b, bits >> 31 ? bits : ~bits & 0x7fffffffu, min(max(__float_as_int(x[K]), 0), p.vocab - 1));
        return kind[b] == 1 ? (double)v - highest[b] - log_sum[b] + base[b] : -INFINITY;
    };
    auto take = [&](int i, double v, BeamKey at) {
        const int b = (int)(at >> 60), w = (int)(at & 0xfffffffu);
        token[i] = w;
        parent[i] = vb * K + b;
        score_out[i] = (float)v;
        live_out[i] = kind[b] == 1 && w != p.eos;
    };
    // K first entries reach the line: only lists whose first entries do are looked into
    const double own = tid < K && kind[tid] == 2 ? (double)score[tid] : -INFINITY;
    double top = own;
    BeamKey at;
    const BeamKey own_at = key_of(tid & 15, 0, p.eos);           // (its beam's only candidate)
    for (int c = tid; c < lists; c += kThreads) {
        heads[c] = entry(c, 0, &at);
        top = fmax(top, heads[c]);
    }
    if (tid == 0) *walked = 0;
    const double line = block_line(K, s, top);
    for (int c = tid; c < lists; c += kThreads)
        if (heads[c] >= line && heads[c] > -INFINITY) which[atomicAdd(walked, 1)] = c;
    __syncthreads();
    const int entries = *walked * K;
    block_collect(s, [&](auto f) {
#pragma unroll 2
        for (int c = tid; c < entries; c += kThreads) {
            const int list = c / K;
            const double v = entry(which[list], c - list * K, &at);
            if (v >= line) f(v, at);
        }
        if (own >= line) f(own, own_at);
    });
    __syncthreads();
    const int n = s.count;
    const int found = n <= kBeamRoom ? block_place(K, s, n, take) : block_top(K, s,
        [&](auto f) {
            for (int c = tid; c < lists * K; c += kThreads) {
                const int list = c / K;
                const double v = entry(list, c - list * K, &at);
                f(v, at);
            }
            f(own, own_at);
        }, take);
    if (tid >= found && tid < K) {
        token[tid] = -1;
        parent[tid] = -1;
        score_out[tid] = -INFINITY;
        live_out[tid] = 0;
    }
    return true;
}

}  // namespace reef
