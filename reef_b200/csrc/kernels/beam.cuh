// Beam search's selection: of every request the `beams` best continuations over its beams and the vocabulary,
//   cand(b, w) = score[b] + logits[b][w] - log sum_u exp(logits[b][u]),
// ties by the lowest b * vocab + w.  A beam that has ended (live 0) competes with its score and the end word alone; candidates of
// -infinity or NaN are none, so a row without a finite sum (a NaN, an infinity, nothing but -infinity) has none, nor has a beam without a
// finite score.  What is missing comes
// out as token -1, parent -1, score -infinity, live 0.
#pragma once
#include "paged_cache.cuh"

namespace reef {

constexpr int kBeamMax = 16;
constexpr int kBeamVecs = 4;                              // 128-bit loads of a lane and turn
constexpr int kBeamTurn = kBeamVecs * 4 * 32;             // words of a warp's turn
constexpr int kBeamRoom = 512;                            // candidates that a block ranks side by side
// Parts of a row of logits, a part to a block: a turn of its eight warps at least, and over all rows not more than four blocks to an SM
// (a second round of blocks repeats what a block has to do once: 256 rows in 2 parts each 39 us, in 4 parts 50, in 1 part 41).
__host__ inline int beam_parts(long long rows, int vocab) {
    const long long least = 8LL * kBeamTurn, most = (vocab + least - 1) / least, slots = 4 * 148;
    if (rows * most <= slots) return (int)most;
    if (rows <= slots) return (int)(slots / rows);
    return 1;
}
__host__ __device__ inline int beam_part_floats(int beams) { return 2 + 2 * beams; }

template <class V>
struct BeamRoom {
    V value[kBeamRoom];
    int index[kBeamRoom];
    V line[8];
    int who[8];
    int count;
};
constexpr int kBeamSmem = (int)sizeof(BeamRoom<double>);

template <class V>
__device__ __forceinline__ bool beam_before(V a, int ia, V b, int ib) { return a > b || (a == b && ia < ib); }

// The K greatest of all threads' values in their order, ties by the lowest index; `each(f)` calls f(value, index) for those of this
// thread, -infinity and NaN are none.  Every warp's K-th greatest of its lanes' maxima has K values at or above it, so the greatest of
// these eight is a line that few values reach: those are ranked against each other.  Where more reach it than there is room (many equal
// values) the best one behind the last is looked for K times.  `take(i, value, index)` gets the i-th; returns how many there are.
template <class V, class Each, class Take>
__device__ __forceinline__ int block_top(int K, BeamRoom<V>& s, Each each, Take take) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const V ninf = -INFINITY;
    V top = ninf;
    each([&](V v, int) { if (v > top) top = v; });
    int rank = 0;
#pragma unroll
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
    each([&](V v, int i) {
        if (v >= line && v > ninf) {
            const int at = atomicAdd(&s.count, 1);
            if (at < kBeamRoom) {
                s.value[at] = v;
                s.index[at] = i;
            }
        }
    });
    __syncthreads();
    const int n = s.count;
    if (n <= kBeamRoom) {
        for (int c = tid; c < n; c += kThreads) {
            const V v = s.value[c];
            const int i = s.index[c];
            int r = 0;
            for (int o = 0; o < n && r < K; o++) r += beam_before(s.value[o], s.index[o], v, i);
            if (r < K) take(r, v, i);
        }
        return min(n, K);
    }
    V last = INFINITY;
    int last_i = -1, found = 0;
    for (; found < K; found++) {
        V best = ninf;
        int best_i = 0x7fffffff;
        each([&](V v, int i) {
            if (v > ninf && beam_before(last, last_i, v, i) && beam_before(v, i, best, best_i)) best = v, best_i = i;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const V v = __shfl_xor_sync(0xffffffffu, best, o);
            const int i = __shfl_xor_sync(0xffffffffu, best_i, o);
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
// args: logits, live, [start], parts.  One pass, a range of the part to a warp, no warp waiting for another until the end: a lane carries a
// maximum and a sum of its own, the next turn's loads are under way while a turn is looked at.  The greatest words so far stand in their
// order in the warp's first K lanes; a word that is greater than the last of them moves in by a shuffle.  What keeps that rare: the first
// turn begins with the K-th greatest of the lanes' maxima as a line, and the greatest line of the block's warps holds for all of them.
// HBM, or L2 where the projection has just left the logits, would bound it; what does are instructions: 256 rows of 100003 words, 95 MB, 39 us (0.37 of the measured copy rate), 61 with a room in shared memory that was
// ranked whenever it filled; four rows of 30522 words 8.
struct BeamScan {
    float value[8][kBeamMax];
    int index[8][kBeamMax];
    float top[8], sum[8];
    float line;                  // K words of the part are at or above it
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
    auto load = [&](float4 (&y)[kBeamVecs], int at) {
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++) {
            const int w = at + (i * 32 + lane) * 4;
            if (w >= 0 && w + 4 <= end) {
                y[i] = *reinterpret_cast<const float4*>(logits + w);
            } else {
                float z[4];
#pragma unroll
                for (int e = 0; e < 4; e++) z[e] = w + e >= 0 && w + e < end ? logits[w + e] : -INFINITY;
                y[i] = make_float4(z[0], z[1], z[2], z[3]);
            }
        }
    };
    int here = begin;                          // first word of this turn
    float top = -INFINITY;
    float2 sum = make_float2(0.f, 0.f);
    // this lane's word among the K greatest; the last of them
    float mine = -INFINITY, last = -INFINITY;
    int mine_i = 0x7fffffff, last_i = 0x7fffffff;
    auto move_in = [&](float v, int w) {       // (the same v and w in all lanes; it comes before the last)
        const int at = __popc(__ballot_sync(0xffffffffu, lane < K && beam_before(mine, mine_i, v, w)));
        const float pv = __shfl_up_sync(0xffffffffu, mine, 1);
        const int pi = __shfl_up_sync(0xffffffffu, mine_i, 1);
        if (lane >= at) {
            mine = lane == at ? v : pv;
            mine_i = lane == at ? w : pi;
        }
        last = __shfl_sync(0xffffffffu, mine, K - 1);
        last_i = __shfl_sync(0xffffffffu, mine_i, K - 1);
    };
    // the greatest line of the block's warps: as an integer a float >= 0 keeps its order, a float < 0 has it turned round
    auto raise = [&](float v) {
        if (v >= 0.f) atomicMax((int*)&s.line, __float_as_int(v));
        else atomicMin((unsigned*)&s.line, __float_as_uint(v));
    };
    bool stopped = false;
    int up = 0, turns = 0;
    load(x, begin);
    __syncthreads();                           // a persistent caller's previous block is out of shared memory
    if (tid == 0) s.line = -INFINITY;
    __syncthreads();
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
        float h[kBeamVecs];
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++) h[i] = fmaxf(fmaxf(x[i].x, x[i].y), fmaxf(x[i].z, x[i].w));
        const float high = fmaxf(fmaxf(h[0], h[1]), fmaxf(h[2], h[3]));
        if (high > top) {
            const float by = exp2_fast((top - high) * kLog2e);
            sum.x *= by;
            sum.y *= by;
            top = high;
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
        float line = *(volatile float*)&s.line;        // nothing below it counts, in this warp or another
        if (here == begin) {
            int rank = 0;
#pragma unroll
            for (int j = 0; j < 32; j++) {
                const float v = __shfl_sync(0xffffffffu, high, j);
                rank += v > high || (v == high && j < lane);
            }
            line = fmaxf(line, __shfl_sync(0xffffffffu, high, __ffs(__ballot_sync(0xffffffffu, rank == K - 1)) - 1));
        }
        // (an equal word of this warp's later turns is too late; among one turn's, and another warp's, it need not be)
        auto counts = [&](float v, int w) { return v >= line && v > -INFINITY && beam_before(v, w, last, last_i); };
        if (__any_sync(0xffffffffu, high >= line && high > -INFINITY && high >= last)) {
            const float before = last;
#pragma unroll
            for (int i = 0; i < kBeamVecs; i++) {
                if (!__any_sync(0xffffffffu, h[i] >= line && h[i] >= last)) continue;
                const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                const int w = here + (i * 32 + lane) * 4;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    unsigned m = __ballot_sync(0xffffffffu, counts(v[e], w + e));
                    while (m) {
                        const int src = __ffs(m) - 1;
                        move_in(__shfl_sync(0xffffffffu, v[e], src), __shfl_sync(0xffffffffu, w + e, src));
                        m &= m - 1;
                        m &= __ballot_sync(0xffffffffu, counts(v[e], w + e));
                    }
                }
            }
            if (lane == 0 && last > before && last > line) raise(last);
        }
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++) x[i] = next[i];
    }
    // the warps' sums and candidates meet
    float high = warp_max(top);
    const float part_sum = sum.x + sum.y, total = warp_sum(top == -INFINITY ? part_sum : part_sum * exp2_fast((top - high) * kLog2e));
    if (lane == 0) {
        s.top[warp] = high;
        s.sum[warp] = total;
    }
    if (lane < K) {
        s.value[warp][lane] = mine;
        s.index[warp][lane] = mine_i;
    }
    if (__syncthreads_or(stopped)) return false;
    if (tid == 0) {
        float all = 0.f;
        for (int w = 0; w < 8; w++) high = fmaxf(high, s.top[w]);
        for (int w = 0; w < 8; w++) all += s.top[w] == -INFINITY ? s.sum[w] : s.sum[w] * exp2_fast((s.top[w] - high) * kLog2e);
        out[0] = high;
        out[1] = all;
    }
    if (tid < 8 * K) {
        // a candidate's place: how many come before it; those that are none stand behind them, the lowest first
        const int w = tid / K, c = tid - w * K, index = s.index[w][c];
        const float v = s.value[w][c];
        int at = 0;
#pragma unroll
        for (int o = 0; o < 8; o++)
            for (int k = 0; k < K; k++) {
                const float u = s.value[o][k];
                const int i = s.index[o][k];
                at += beam_before(u, i, v, index) || (u == v && i == index && o * K + k < tid);
            }
        if (at < K) {
            out[2 + at] = v;
            out[2 + K + at] = __int_as_float(index);
        }
    }
    return true;
}

// ---- pick: the parts of a request's beams -> its new beams --------------------------------------------------------------------
// args: parts, score, live, [start], token, parent, score', live'.  Within a beam the logits decide, exactly as they are; beams are
// compared in 64 bits: a score of -50 in 32 bits cannot tell logits apart that differ by less than 4e-6.  Latency: 32 requests of eight beams
// 8 us.
__host__ inline int beam_pick_smem() { return kBeamSmem + kBeamMax * (8 + 8 + 4 + 4); }
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
    BeamRoom<double>& s = *reinterpret_cast<BeamRoom<double>*>(smem);
    // of a beam: its logits' maximum, the logarithm of the sum of exponentials below it, its score.  Applied one after the other: their sum
    // would lose the smaller ones where the logits are at the type's lowest value.
    double* log_sum = reinterpret_cast<double*>(smem + kBeamSmem);
    double* base = log_sum + kBeamMax;
    float* highest = reinterpret_cast<float*>(base + kBeamMax);
    int* kind = reinterpret_cast<int*>(highest + kBeamMax);           // 0: no candidates, 1: its parts, 2: it has ended
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
    const int lists = K * p.parts;
    const int found = block_top<double>(K, s,
        [&](auto f) {
            for (int c = tid; c < lists; c += kThreads) {
                const int b = c / p.parts;
                if (kind[b] != 1) continue;
                const float* x = parts + (size_t)c * F;
                for (int i = 0; i < K; i++) {
                    const float v = x[2 + i];
                    const int w = __float_as_int(x[2 + K + i]);
                    if (v == -INFINITY) break;
                    f((double)v - highest[b] - log_sum[b] + base[b], b * p.vocab + min(max(w, 0), p.vocab - 1));
                }
            }
            if (tid < K && kind[tid] == 2) f((double)score[tid], tid * p.vocab + p.eos);
        },
        [&](int i, double v, int at) {
            const int b = at / p.vocab, w = at - b * p.vocab;
            token[i] = w;
            parent[i] = vb * K + b;
            score_out[i] = (float)v;
            live_out[i] = kind[b] == 1 && w != p.eos;
        });
    if (tid >= found && tid < K) {
        token[tid] = -1;
        parent[tid] = -1;
        score_out[tid] = -INFINITY;
        live_out[tid] = 0;
    }
    return true;
}

}  // namespace reef
