// Beam search's selection: of every request the `beams` best continuations over its beams and the vocabulary,
//   cand(b, w) = score[b] + logits[b][w] - log sum_u exp(logits[b][u]),
// ties by the lowest b * vocab + w.  A beam that has ended (live 0) competes with its score and the end word alone; candidates of
// -infinity or NaN are none, so a row without a finite sum (a NaN, an infinity, nothing but -infinity) has none, nor has a beam without a
// finite score.  What is missing comes
// out as token -1, parent -1, score -infinity, live 0.
#pragma once
#include "simple.cuh"

namespace reef {

constexpr int kBeamMax = 16;
constexpr int kBeamVecs = 4;                              // 128-bit loads of a thread and turn
constexpr int kBeamTurn = kBeamVecs * 4 * kThreads;       // words of a turn
constexpr int kBeamRoom = 512;                            // candidates that are ranked side by side
// Parts of a row of logits: four blocks to an SM over all rows, a turn to a part at least.
__host__ inline int beam_parts(long long rows, int vocab) {
    const long long turns = ((vocab + 3LL) / 4 + 1 + kBeamTurn / 4 - 1) / (kBeamTurn / 4), want = (4 * 148 + rows - 1) / rows;
    return (int)(turns < want ? turns : want);
}
__host__ __device__ inline int beam_part_floats(int beams) { return 2 + 2 * beams; }

template <class V>
struct BeamRoom {
    V value[kBeamRoom];
    int index[kBeamRoom];
    V line[8];
    int who[8];
    V best[2 * kBeamMax];
    int best_index[2 * kBeamMax];
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
// args: logits, live, [start], parts.  One pass: a thread carries a maximum and a sum of its own, the next turn's loads are under way while
// a turn is looked at.  The first turn gives a line below which nothing counts any more; later turns add the few words above it
// (words come in their order, so an equal one is too late), the line rises whenever the room is half full.  Bound by HBM (or L2, where the
// projection has just left the logits).
__device__ __forceinline__ bool body_beam_scan(const KTask& t, int vb, unsigned char* smem, const int* flag) {
    const BeamP& p = t.p.beam;
    const int r = vb / p.parts, part = vb - r * p.parts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.beams;
    const int* live = (const int*)t.a[1];
    const int* start = p.has_start ? (const int*)t.a[2] : nullptr;
    float* out = (float*)t.a[2 + p.has_start] + (size_t)vb * beam_part_floats(K);
    if (live[r] == 0) return true;
    const int row = beam_logits(p, start, r);
    if (row < 0) return true;
    BeamRoom<float>& s = *reinterpret_cast<BeamRoom<float>*>(smem);
    // loads begin at a 16-byte boundary: up to three words of the row before are masked
    const float* logits = (const float*)t.a[0] + (size_t)row * p.vocab;
    const int lead = (int)(((size_t)row * p.vocab) & 3);
    const int begin = part * p.part * 4 - lead, end = min(p.vocab, begin + p.part * 4);
    float x[kBeamVecs][4], next[kBeamVecs][4];
    auto word = [&](int at, int i) { return at + (i * kThreads + tid) * 4; };        // first word of a load
    auto load = [&](float (&y)[kBeamVecs][4], int at) {
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++) {
            const int w = word(at, i);
            if (w >= 0 && w + 4 <= end) {
                const float4 v = *reinterpret_cast<const float4*>(logits + w);
                y[i][0] = v.x; y[i][1] = v.y; y[i][2] = v.z; y[i][3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) y[i][e] = w + e >= 0 && w + e < end ? logits[w + e] : -INFINITY;
            }
        }
    };
    float top = -INFINITY, sum = 0.f, line = -INFINITY;
    int here = begin, up = 0, have = 0;        // first word of this turn; candidates in the room
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) f(x[i][e], word(here, i) + e);
    };
    // the K greatest of the room's `count` go to its front, in their order
    auto rank = [&](int count) {
        float v[kBeamRoom / kThreads];
        int w[kBeamRoom / kThreads], at[kBeamRoom / kThreads];
#pragma unroll
        for (int i = 0; i < kBeamRoom / kThreads; i++) {
            const int c = tid + i * kThreads;
            at[i] = K;
            if (c < count) {
                v[i] = s.value[c];
                w[i] = s.index[c];
                at[i] = 0;
                for (int o = 0; o < count && at[i] < K; o++) at[i] += beam_before(s.value[o], s.index[o], v[i], w[i]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kBeamRoom / kThreads; i++)
            if (at[i] < K) {
                s.value[at[i]] = v[i];
                s.index[at[i]] = w[i];
            }
        if (tid == 0) s.count = min(count, K);
        __syncthreads();
        if (count >= K) line = s.value[K - 1];
        return min(count, K);
    };
    load(x, begin);
    __syncthreads();                           // a persistent caller's previous block is out of shared memory
    for (; here < end; here += kBeamTurn) {
        if (flag != nullptr) {                 // best-effort flavour: a look at the preempt flag, asked for a turn ahead
            if (__syncthreads_or(up)) return false;
            up = tid == 0 ? ld_flag(flag) : 0;
        }
        if (here + kBeamTurn < end) load(next, here + kBeamTurn);
        float high = top;
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++) high = fmaxf(fmaxf(fmaxf(high, x[i][0]), fmaxf(x[i][1], x[i][2])), x[i][3]);
        if (high > top) {
            sum *= __expf(top - high);
            top = high;
        }
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum += x[i][e] == -INFINITY ? 0.f : __expf(x[i][e] - top);
        if (here == begin) {
            have = block_top<float>(K, s, each, [&](int i, float v, int w) { s.best[i] = v; s.best_index[i] = w; });
            __syncthreads();
            if (tid < have) {
                s.value[tid] = s.best[tid];
                s.index[tid] = s.best_index[tid];
            }
            if (tid == 0) s.count = have;
            if (have == K) line = s.best[K - 1];
            __syncthreads();
        } else {
            each([&](float v, int w) {
                if (v > line) {
                    const int at = atomicAdd(&s.count, 1);
                    if (at < kBeamRoom) {
                        s.value[at] = v;
                        s.index[at] = w;
                    }
                }
            });
            __syncthreads();
            const int count = s.count;
            __syncthreads();
            if (count > kBeamRoom) {
                // more than there is room for: what was there before, this turn by itself, and the two together
                have = rank(have);
                if (tid < have) {
                    s.best[tid] = s.value[tid];
                    s.best_index[tid] = s.index[tid];
                }
                __syncthreads();
                const int found = block_top<float>(K, s, each, [&](int i, float v, int w) { s.best[have + i] = v; s.best_index[have + i] = w; });
                __syncthreads();
                have += found;
                if (tid < have) {
                    s.value[tid] = s.best[tid];
                    s.index[tid] = s.best_index[tid];
                }
                __syncthreads();
                have = rank(have);
            } else {
                have = count > kBeamRoom / 2 ? rank(count) : count;
            }
        }
#pragma unroll
        for (int i = 0; i < kBeamVecs; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[i][e] = next[i][e];
    }
    have = rank(have);
    if (tid < K) {
        out[2 + tid] = tid < have ? s.value[tid] : -INFINITY;
        out[2 + K + tid] = __int_as_float(tid < have ? s.index[tid] : 0);
    }
    // all threads' sums
    float high = warp_max(top);
    if (lane == 0) s.line[warp] = high;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) high = fmaxf(high, s.line[w]);
    sum = warp_sum(top == -INFINITY ? sum : sum * __expf(top - high));
    if (lane == 0) s.best[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 8; w++) sum += s.best[w];
        out[0] = high;
        out[1] = sum;
    }
    return true;
}

// ---- pick: the parts of a request's beams -> its new beams --------------------------------------------------------------------
// args: parts, score, live, [start], token, parent, score', live'.  Within a beam the logits decide, exactly as they are; beams are
// compared in 64 bits: a score of -50 in 32 bits cannot tell logits apart that differ by less than 4e-6.
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
