// g4_beam.cu — beam search's selection over beams and vocabulary.
//
// Within a row (beam) log softmax keeps the order of the logits, so a row's
// `beams` best candidates are its `beams` largest logits, and one pass over the
// logits gives them and the softmax's sum:
//   k_beam_rows   one CTA per slice of a row: max, sum of exp, the slice's best
//   k_beam_merge  one CTA per group: the rows' sums, scores, the group's best
// The logits are read once and HBM bounds the pass: each thread holds its
// values in registers for all three results.
#include <cuda_runtime.h>
#include <math.h>

#include "g4_kv4.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kOcc = 4;             // CTAs per SM: 64 KB of loads in flight
constexpr int kChunk = 4096;        // values that a CTA holds in registers at a time
constexpr int kMaxBeams = 32;
constexpr int kMergeThreads = 512;
constexpr int kBuffer = 512;       // candidates above the threshold of one CTA
constexpr float kC = 1.4426950408889634f;

// (value, index) as one number, larger = better: a larger value, then a lower
// index. -0 and +0 are one value; NaN counts as -inf.
G4_DEV uint32_t order_f32(float x) {
    const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
G4_DEV float value_f32(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
G4_DEV uint64_t key_of(float x, uint32_t i) { return (uint64_t)order_f32(x) << 32 | (uint32_t)~i; }

// What a slice leaves: max, sum of its exponentials, then `beams` keys, best first
// (0: the slice has no more values).
struct SliceStat {
    float max;
    double sum;      // of e^(x - max)
};

struct BeamArgs {
    const void *logits;
    long long stride;
    int vocab, beams, slices, chunks;      // slices per row, chunks per slice
    SliceStat *stats;                    // [rows][slices]
    uint64_t *keys;                      // [rows][slices][beams]
    const float *scores;
    const unsigned char *finished;
    int eos;
    float *out_scores;
    int *parents, *tokens;
    unsigned char *out_finished;
};

template <typename T>
struct Wide;    // 16 bytes of values
template <>
struct Wide<float> {
    static constexpr int N = 4;
    static G4_DEV void get(const uint4 &w, float *x) {
        x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y);
        x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
    }
};
template <>
struct Wide<__nv_bfloat16> {
    static constexpr int N = 8;
    static G4_DEV void get(const uint4 &w, float *x) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
};
template <>
struct Wide<__half> {
    static constexpr int N = 8;
    static G4_DEV void get(const uint4 &w, float *x) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&w);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
};

G4_DEV uint64_t warp_max64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
        v = v > w ? v : w;
    }
    return v;
}

G4_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One CTA per slice of a.chunks chunks of kChunk values of a row. VEC: rows start
// on 16 bytes. Each thread keeps a running maximum and sum, the next chunk's loads
// in flight in registers while it works on one; the CTA's threads meet in chunks 0,
// 1, 2, 4, ... for a threshold that few values pass. The pass is bound by its
// instructions (14 a value) as much as by HBM: 128 rows of 262144 in fp32 take 30 us
// (4.5 TB/s), in bf16 the same. Measured beside it (with the merge, 36 us): 32 values a
// thread and chunk 41 us, five CTAs an SM 37 us, two waves of shorter slices 37 us,
// rings of 48 KB in shared memory filled by cp.async 39 us.
// A slice whose first chunk is one value throughout (masked) has that value for its
// threshold: more than kBuffer pass, and the slice is read again for every beam. 16 x 8
// beams of 262144 with the first half masked 343 us; with 99 % masked here and there 37 us
// (-inf) to 43 (-1e10).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, kOcc) k_beam_rows(BeamArgs a) {
    constexpr int N = Wide<T>::N, E = kChunk / kThreads, V = E / N;
    __shared__ uint64_t buf[kBuffer];
    __shared__ float gmax[2][32];
    __shared__ float wmax[kThreads / 32];
    __shared__ double wsum[kThreads / 32];
    __shared__ uint64_t wkey[kThreads / 32];
    __shared__ int count;
    griddep_wait();
    griddep_launch();
    const int row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *p = reinterpret_cast<const T *>(a.logits) + row * a.stride;
    const int first = slice * a.chunks * kChunk, end = min(a.vocab, first + a.chunks * kChunk);
    // value e of this thread in the chunk at `base`
    auto index = [&](int base, int e) { return base + (e / N) * (kThreads * N) + tid * N + e % N; };
    float x[E];
    auto largest = [&]() {
        float m[4];
#pragma unroll
        for (int e = 0; e < 4; e++) m[e] = x[e];
#pragma unroll
        for (int e = 4; e < E; e++) m[e & 3] = fmaxf(m[e & 3], x[e]);
        return fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), -INFINITY);      // NaN: none
    };
    // Up to kFar the sum is of 2^(c x - m2), one fma a value, with c = log2 e rounded to fp32
    // and m2 = c tmax, rounded: at most 16 off, and put right when the threads join. A
    // larger maximum (a mask of -1e10 or of the type's lowest value wherever no token of
    // the thread is left) would make that factor overflow, or m2 itself: there the sum is of
    // 2^(c (x - tmax)).
    constexpr float kFar = 0x1p28f;
    float tmax = -INFINITY, m2 = 0.0f, sum = 0.0f;
    auto near = [&](float m) { return fabsf(m) <= kFar; };
    auto off = [&](float m, float c2) { return near(m) ? fmaf(-kC, m, c2) : 0.0f; };      // m2 - c m
    auto add = [&](float m) {
        if (m > tmax) {
            const float n2 = m * kC;
            if (near(tmax) && near(m)) sum *= ex2(m2 - n2);
            else if (tmax > -INFINITY) sum *= ex2(fmaf(tmax - m, kC, off(tmax, m2) - off(m, n2)));
            tmax = m;
            m2 = n2;
        }
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (near(tmax)) {
#pragma unroll
            for (int e = 0; e < E; e++) part[e & 3] += ex2(fmaf(x[e], kC, -m2));
        } else if (tmax > -INFINITY) {
#pragma unroll
            for (int e = 0; e < E; e++) part[e & 3] += ex2((x[e] - tmax) * kC);
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
    };
    // the maxima of 32 groups of threads: the k-th largest is a threshold that at
    // least k values reach
    float tau;
    auto threshold = [&](float m, int parity) {
        constexpr int kPerGroup = kThreads / 32;
#pragma unroll
        for (int o = kPerGroup / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (tid % kPerGroup == 0) gmax[parity][tid / kPerGroup] = m;
        __syncthreads();
        // every warp ranks the 32 for itself: no second barrier (and the buffers alternate)
        const float g = gmax[parity][lane];
        int rank = 0;
#pragma unroll
        for (int o = 0; o < 32; o++) {
            const float other = gmax[parity][o];
            rank += (int)(other > g) + ((int)(other == g) & (int)(o < lane));
        }
        tau = __shfl_sync(0xffffffffu, g, __ffs(__ballot_sync(0xffffffffu, rank == a.beams - 1)) - 1);
    };
    auto collect = [&](int base, float m) {
        if (m >= tau) {                                    // NaN is a candidate only if tau is -inf
            uint32_t hit = 0;
#pragma unroll
            for (int e = 0; e < E; e++) hit |= x[e] < tau ? 0u : 1u << e;
            while (hit) {
                const int at_e = __ffs(hit) - 1, i = index(base, at_e);
                hit &= hit - 1;
                float y = x[0];
#pragma unroll
                for (int e = 1; e < E; e++) y = e == at_e ? x[e] : y;
                if (i < end) {
                    const int at = atomicAdd(&count, 1);
                    if (at < kBuffer) buf[at] = key_of(y, i);
                }
            }
        }
    };

    int round = 0, parity = 0;
    auto work = [&](int base) {
        const float m = largest();
        add(m);
        if ((round & (round - 1)) == 0) threshold(tmax, parity ^= 1);      // chunks 0, 1, 2, 4, 8, ...
        collect(base, m);
        round++;
    };
    if (tid == 0) count = 0;
    int base = first;
    if (VEC) {
        const uint4 *q = reinterpret_cast<const uint4 *>(p + first) + tid;
        uint4 u[V], w[V];
        auto fetch = [&](uint4 (&to)[V], int chunk) {
#pragma unroll
            for (int v = 0; v < V; v++) to[v] = __ldcs(q + (long long)chunk * (kChunk / N) + v * kThreads);
        };
        auto take = [&](const uint4 (&from)[V]) {
#pragma unroll
            for (int v = 0; v < V; v++) Wide<T>::get(from[v], x + v * N);
        };
        const int full = (end - first) / kChunk;
        if (full > 0) fetch(u, 0);
        for (int c = 0; c < full; c += 2) {
            if (c + 1 < full) fetch(w, c + 1);
            take(u);
            work(base);
            base += kChunk;
            if (c + 1 < full) {
                if (c + 2 < full) fetch(u, c + 2);
                take(w);
                work(base);
                base += kChunk;
            }
        }
    }
    for (; base < end; base += kChunk) {                   // a part of a chunk, or rows that start anywhere
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int i = index(base, e);
            x[e] = i < end ? (float)p[i] : -INFINITY;
        }
        work(base);
    }
    if (sum != sum) {                                      // a NaN among the values is not a token: once more without
        sum = 0.0f;
        for (base = first; base < end; base += kChunk)
            for (int e = 0; e < E; e++) {
                const int i = index(base, e);
                const float y = i < end ? (float)p[i] : -INFINITY;
                if (y == y) sum += ex2(near(tmax) ? fmaf(y, kC, -m2) : (y - tmax) * kC);
            }
    }

    // the slice's sum: per thread in fp32, over threads in fp64
    float bm = warp_max(tmax);
    if (lane == 0) wmax[warp] = bm;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; i++) bm = fmaxf(bm, wmax[i]);
    double total = tmax == -INFINITY ? 0.0 : (double)sum * (double)ex2(fmaf(tmax - bm, kC, off(tmax, m2)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) wsum[warp] = total;
    __syncthreads();
    if (tid == 0) {
        double all = 0.0;
        for (int i = 0; i < kThreads / 32; i++) all += wsum[i];
        a.stats[(long long)row * a.slices + slice] = {bm, all};
    }
    const int n = count;
    uint64_t *out = a.keys + ((long long)row * a.slices + slice) * a.beams;
    if (n <= kBuffer) {
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t mine = buf[i];
            int rank = 0;
            for (int j = 0; j < n; j++) rank += buf[j] > mine;
            if (rank < a.beams) out[rank] = mine;
        }
        for (int i = n + tid; i < a.beams; i += kThreads) out[i] = 0;
        return;
    }
    // more equal or rising values than the buffer holds: one round per candidate
    uint64_t below = ~0ull;
    for (int r = 0; r < a.beams; r++) {
        uint64_t best = 0;
        for (int i = first + tid; i < end; i += kThreads) {
            const uint64_t k = key_of((float)p[i], i);
            if (k < below && k > best) best = k;
        }
        best = warp_max64(best);
        __syncthreads();
        if (lane == 0) wkey[warp] = best;
        __syncthreads();
        best = 0;
        for (int i = 0; i < kThreads / 32; i++) best = wkey[i] > best ? wkey[i] : best;
        if (tid == 0) out[r] = best;
        below = best;
    }
}

// ---- merge ------------------------------------------------------------------
// fp64 scores in the order of unsigned integers; NaN counts as -inf.
G4_DEV uint64_t order_f64(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x != x ? -(double)INFINITY : x + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
G4_DEV double value_f64(uint64_t o) {
    return __longlong_as_double((long long)(o >> 63 ? o & 0x7fffffffffffffffull : ~o));
}

// Candidate c of a group as (order of its score, beam and token): c counts
// the rows' slices' keys; a row that is finished, or whose candidates are all
// -inf, offers its first tokens instead (and the finished one eos).
struct Cand {
    uint64_t score;
    uint64_t at;     // beam << 32 | token, ~0: none
};

G4_DEV bool better(const Cand &x, const Cand &y) {
    return x.at != ~0ull && (y.at == ~0ull || x.score > y.score || (x.score == y.score && x.at < y.at));
}

// One CTA per group. Candidates are few (beams per slice), so the same threshold
// as in a slice leaves little more than `beams` of them, which rank one another.
__global__ void __launch_bounds__(kMergeThreads) k_beam_merge(BeamArgs a) {
    __shared__ double lsum[kMaxBeams];      // of a live row: log of the sum of e^(x - top)
    __shared__ float top[kMaxBeams];
    __shared__ float cums[kMaxBeams];
    __shared__ int kind[kMaxBeams];         // 0 live, 1 all -inf, 2 finished
    __shared__ uint64_t gmax[32], b_score[kBuffer], b_at[kBuffer];
    __shared__ int count;
    griddep_wait();
    const int grp = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) count = 0;
    for (int r = warp; r < a.beams; r += kMergeThreads / 32) {
        const SliceStat *st = a.stats + ((long long)grp * a.beams + r) * a.slices;
        const float cum = a.scores[grp * a.beams + r];
        const bool done = a.finished && a.finished[grp * a.beams + r];
        float m = -INFINITY;
        for (int s = lane; s < a.slices; s += 32) m = fmaxf(m, st[s].max);
        m = warp_max(m);
        double sum = 0.0;
        for (int s = lane; s < a.slices; s += 32)
            if (st[s].max > -INFINITY) sum += st[s].sum * exp((double)st[s].max - (double)m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            cums[r] = cum;
            kind[r] = cum - cum != 0.0f ? 1 : done ? 2 : m - m != 0.0f ? 1 : 0;
            top[r] = m;
            lsum[r] = kind[r] == 0 ? log(sum) : 0.0;
        }
    }
    __syncthreads();
    const int per_row = a.slices * a.beams + 1, total = a.beams * per_row, few = min(a.beams, a.vocab);
    auto cand = [&](int c) -> Cand {
        const int r = (int)((unsigned)c / (unsigned)per_row), j = c - r * per_row;
        Cand x = {0, ~0ull};
        if (kind[r] == 0) {
            const uint64_t key = j < per_row - 1 ? a.keys[((long long)grp * a.beams + r) * a.slices * a.beams + j] : 0;
            if (key) {
                // (the maximum first: beside one of 1e10 the logarithm would be lost)
                x.score = order_f64((double)cums[r] +
                                    (((double)value_f32((uint32_t)(key >> 32)) - (double)top[r]) - lsum[r]));
                x.at = (uint64_t)r << 32 | (uint32_t)~(uint32_t)key;
            }
        } else if (j < few) {
            x.score = order_f64(kind[r] == 2 && j == a.eos ? (double)cums[r] : -(double)INFINITY);
            x.at = (uint64_t)r << 32 | (uint32_t)j;
        } else if (j == per_row - 1 && kind[r] == 2 && a.eos >= few) {
            x.score = order_f64((double)cums[r]);
            x.at = (uint64_t)r << 32 | (uint32_t)a.eos;
        }
        return x;
    };
    auto put = [&](int k, const Cand &x) {
        const int o = grp * a.beams + k, r = (int)(x.at >> 32), tok = (int)(uint32_t)x.at;
        a.out_scores[o] = (float)value_f64(x.score);
        a.parents[o] = r;
        a.tokens[o] = tok;
        if (a.out_finished) a.out_finished[o] = (a.finished && a.finished[grp * a.beams + r]) || tok == a.eos;
    };
    // maxima of 32 groups of threads (0: none; the order of any score is larger)
    uint64_t hm = 0;
    for (int c = tid; c < total; c += kMergeThreads) {
        const Cand x = cand(c);
        if (x.at != ~0ull && x.score > hm) hm = x.score;
    }
    constexpr int kPerGroup = kMergeThreads / 32;
#pragma unroll
    for (int o = kPerGroup / 2; o > 0; o >>= 1) {
        const uint64_t y = __shfl_xor_sync(0xffffffffu, hm, o);
        hm = y > hm ? y : hm;
    }
    if (tid % kPerGroup == 0) gmax[tid / kPerGroup] = hm;
    __syncthreads();
    const uint64_t g = gmax[lane];
    int rank = 0;
#pragma unroll
    for (int o = 0; o < 32; o++) {
        const uint64_t other = gmax[o];
        rank += (int)(other > g) + ((int)(other == g) & (int)(o < lane));
    }
    const uint64_t tau = __shfl_sync(0xffffffffu, g, __ffs(__ballot_sync(0xffffffffu, rank == a.beams - 1)) - 1);
    for (int c = tid; c < total; c += kMergeThreads) {
        const Cand x = cand(c);
        if (x.at != ~0ull && x.score >= tau) {
            const int at = atomicAdd(&count, 1);
            if (at < kBuffer) {
                b_score[at] = x.score;
                b_at[at] = x.at;
            }
        }
    }
    __syncthreads();
    const int n = count;
    if (n <= kBuffer) {
        for (int i = tid; i < n; i += kMergeThreads) {
            const Cand x = {b_score[i], b_at[i]};
            int rank = 0;
            for (int j = 0; j < n; j++) rank += better({b_score[j], b_at[j]}, x);
            if (rank < a.beams) put(rank, x);
        }
        return;
    }
    // more equal candidates than the buffer holds: one round each
    Cand last = {~0ull, 0};
    for (int k = 0; k < a.beams; k++) {
        Cand best = {0, ~0ull};
        for (int c = tid; c < total; c += kMergeThreads) {
            const Cand x = cand(c);
            if (x.at != ~0ull && (k == 0 || better(last, x)) && better(x, best)) best = x;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Cand y = {__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.at, o)};
            if (better(y, best)) best = y;
        }
        __syncthreads();
        if (lane == 0) {
            b_score[warp] = best.score;
            b_at[warp] = best.at;
        }
        __syncthreads();
        best = {b_score[0], b_at[0]};
        for (int w = 1; w < kMergeThreads / 32; w++) {
            const Cand y = {b_score[w], b_at[w]};
            if (better(y, best)) best = y;
        }
        last = best;
        if (tid == 0) put(k, best);
    }
}

// Chunks per slice: as many as give every SM its kOcc CTAs, so that one user's few
// rows spread over the GPU (4 rows of 262144: one chunk each) and many rows run
// in one wave with few slices to join (128 rows: 4 slices each).
constexpr int kSms = 148;
int chunks_per_slice(long long rows, int vocab) {
    const long long chunks = (vocab + kChunk - 1) / kChunk;
    const long long slices = (kOcc * kSms) / rows;                  // per row, in one wave
    return (int)(slices <= 1 ? chunks : (chunks + slices - 1) / slices);
}
int slices_per_row(long long rows, int vocab) {
    const long long slice = (long long)chunks_per_slice(rows, vocab) * kChunk;
    return (int)((vocab + slice - 1) / slice);
}

bool sizes_ok(int groups, int beams, int vocab) {
    return groups >= 0 && groups <= 65536 && beams >= 1 && beams <= kMaxBeams && vocab >= 1 && vocab <= 1 << 24;
}

template <typename T>
cudaError_t launch_rows(const BeamArgs &a, long long rows, cudaStream_t st) {
    const dim3 grid((unsigned)(rows * a.slices)), block(kThreads);
    const bool vec = ((uintptr_t)a.logits & 15) == 0 && a.stride * sizeof(T) % 16 == 0;
    return vec ? g4_launch(k_beam_rows<T, true>, grid, block, 0, st, true, a)
               : g4_launch(k_beam_rows<T, false>, grid, block, 0, st, true, a);
}

}  // namespace

extern "C" {

uint64_t g4_beam_workspace(int groups, int beams, int vocab) {
    if (!sizes_ok(groups, beams, vocab)) return 0;
    // What the largest of all calls of at most these sizes takes: rows that are split have at
    // most kOcc * kSms slices together (of 100000 values, 64 rows have 576 and 128 rows 512).
    const uint64_t rows = (uint64_t)(groups ? groups : 1) * beams, chunks = ((uint64_t)vocab + kChunk - 1) / kChunk,
                   split = rows * chunks < kOcc * kSms ? rows * chunks : kOcc * kSms;
    return (rows > split ? rows : split) * (sizeof(SliceStat) + beams * sizeof(uint64_t));
}

int g4_beam_select(int groups, int beams, int vocab, int type, const void *logits, int64_t logits_stride,
                   const float *scores, const unsigned char *finished, int eos, float *out_scores, int *parents,
                   int *tokens, unsigned char *out_finished, void *workspace, uint64_t workspace_bytes, void *stream) {
    if (!sizes_ok(groups, beams, vocab)) return G4_ERR_INVALID;
    if (type != G4_TYPE_F32 && type != G4_TYPE_BF16 && type != G4_TYPE_F16) return G4_ERR_INVALID;
    if (!logits || !scores || !out_scores || !parents || !tokens || !workspace) return G4_ERR_INVALID;
    if ((uintptr_t)logits % kv4_type_bytes(type) || logits_stride < vocab || logits_stride > (int64_t)1 << 40)
        return G4_ERR_INVALID;
    if (((uintptr_t)scores | (uintptr_t)out_scores | (uintptr_t)parents | (uintptr_t)tokens) & 3)
        return G4_ERR_INVALID;
    if (eos >= vocab || (eos < 0 && finished)) return G4_ERR_INVALID;
    if (((uintptr_t)workspace & 15) || workspace_bytes < g4_beam_workspace(groups, beams, vocab))
        return G4_ERR_INVALID;
    // a group's CTA reads scores and flags while others, and its own threads, write theirs
    const size_t n = (size_t)groups * beams;
    const struct { const void *p; size_t n; } out[4] = {{out_scores, 4 * n}, {parents, 4 * n}, {tokens, 4 * n}, {out_finished, n}};
    for (const auto &x : out)
        if (kv4_overlap(x.p, x.n, scores, 4 * n) || kv4_overlap(x.p, x.n, finished, n)) return G4_ERR_INVALID;
    if (groups == 0) return G4_OK;
    DeviceOf dev(logits);
    if (dev.status() != G4_OK) return dev.status();
    if (!dev.holds(scores) || !dev.holds(finished) || !dev.holds(out_scores) || !dev.holds(parents) ||
        !dev.holds(tokens) || !dev.holds(out_finished) || !dev.holds(workspace))
        return G4_ERR_INVALID;
    BeamArgs a;
    const long long rows = (long long)groups * beams;
    a.logits = logits;
    a.stride = logits_stride;
    a.vocab = vocab;
    a.beams = beams;
    a.chunks = chunks_per_slice(rows, vocab);
    a.slices = slices_per_row(rows, vocab);
    a.keys = (uint64_t *)workspace;
    a.stats = (SliceStat *)(a.keys + rows * a.slices * beams);
    a.scores = scores;
    a.finished = finished;
    a.eos = eos;
    a.out_scores = out_scores;
    a.parents = parents;
    a.tokens = tokens;
    a.out_finished = out_finished;
    const cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (type == G4_TYPE_F32) e = launch_rows<float>(a, rows, st);
    else if (type == G4_TYPE_BF16) e = launch_rows<__nv_bfloat16>(a, rows, st);
    else e = launch_rows<__half>(a, rows, st);
    if (e == cudaSuccess) e = g4_launch(k_beam_merge, dim3(groups), dim3(kMergeThreads), 0, st, true, a);
    return e == cudaSuccess ? G4_OK : G4_ERR_CUDA;
}

}  // extern "C"
