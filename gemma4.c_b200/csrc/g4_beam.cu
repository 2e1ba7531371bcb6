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

constexpr int kThreads = 512;
constexpr int kMaxBeams = 32;
constexpr int kMergeThreads = 256;
constexpr int kBuffer = 1024;      // candidates above the threshold of one CTA

// (value, index) as one number, larger = better: a larger value, then a lower
// index. -0 and +0 are one value; NaN counts as -inf.
G4_DEV uint32_t order_f32(float x) {
    const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
G4_DEV float value_f32(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
G4_DEV uint64_t key_of(float x, uint32_t i) { return (uint64_t)order_f32(x) << 32 | (uint32_t)~i; }

// What a slice leaves: max, sum of exp(x - max), then `beams` keys, best first
// (0: the slice has no more values).
struct SliceStat {
    float max, sum;
};

struct BeamArgs {
    const void *logits;
    long long stride;
    int vocab, beams, slices, slice;     // values per slice
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

// Slice of kThreads * E values, E per thread (a multiple of Wide<T>::N).
// VEC: rows start on 16 bytes.
template <typename T, int E, bool VEC>
__global__ void __launch_bounds__(kThreads) k_beam_rows(BeamArgs a) {
    constexpr int N = Wide<T>::N;
    __shared__ uint64_t buf[kBuffer];
    __shared__ float gmax[32];
    __shared__ double wsum[kThreads / 32];
    __shared__ uint64_t wkey[kThreads / 32];
    __shared__ int count;
    __shared__ uint32_t s_tau;
    griddep_wait();
    const int row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *p = reinterpret_cast<const T *>(a.logits) + row * a.stride;
    const int base = slice * (kThreads * E);
    // value e of this thread is base + (e / N) * kThreads * N + tid * N + e % N
    float x[E];
#pragma unroll
    for (int v = 0; v < E / N; v++) {
        const int i = base + v * (kThreads * N) + tid * N;
        if (VEC && i + N <= a.vocab) {
            const uint4 w = *reinterpret_cast<const uint4 *>(p + i);
            Wide<T>::get(w, x + v * N);
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) x[v * N + j] = i + j < a.vocab ? (float)p[i + j] : -INFINITY;
        }
    }
    if (tid == 0) count = 0;
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; e++) m = fmaxf(m, x[e]);
    // the maxima of the 32 half warps: the k-th largest is a threshold that at
    // least k values reach
    float hm = m;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) hm = fmaxf(hm, __shfl_xor_sync(0xffffffffu, hm, o));
    if ((lane & 15) == 0) gmax[tid >> 4] = hm;
    __syncthreads();
    const float g = gmax[lane];
    float bm = g;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, o));
    if (warp == 0) {
        int rank = 0;
#pragma unroll
        for (int o = 0; o < 32; o++) {
            const float other = __shfl_sync(0xffffffffu, g, o);
            rank += other > g || (other == g && o < lane);
        }
        if (rank == min(a.beams, 32) - 1) s_tau = order_f32(g);
    }
    // sum of exp over the thread's values (pairwise), then over threads in fp64
    const float ref = bm == -INFINITY ? 0.0f : bm;
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < E; e++) part[e & 3] += x[e] == x[e] ? expf(x[e] - ref) : 0.0f;
    double sum = (double)(part[0] + part[1]) + (double)(part[2] + part[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) wsum[warp] = sum;
    __syncthreads();
    const uint32_t tau = s_tau;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const uint32_t o = order_f32(x[e]);
        if (o >= tau) {
            const int i = base + (e / N) * (kThreads * N) + tid * N + e % N;
            if (i < a.vocab) {
                const int at = atomicAdd(&count, 1);
                if (at < kBuffer) buf[at] = (uint64_t)o << 32 | (uint32_t)~i;
            }
        }
    }
    __syncthreads();
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
    } else {
        // more equal values than the buffer holds: one round per candidate
        uint64_t below = ~0ull;
        for (int r = 0; r < a.beams; r++) {
            uint64_t best = 0;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int i = base + (e / N) * (kThreads * N) + tid * N + e % N;
                const uint64_t k = i < a.vocab ? key_of(x[e], i) : 0;
                if (k < below && k > best) best = k;
            }
            best = warp_max64(best);
            __syncthreads();
            if (lane == 0) wkey[warp] = best;
            __syncthreads();
            best = 0;
            for (int w = 0; w < kThreads / 32; w++) best = wkey[w] > best ? wkey[w] : best;
            if (tid == 0) out[r] = best;
            below = best;
        }
    }
    if (tid == 0) {
        double s = 0.0;
        for (int w = 0; w < kThreads / 32; w++) s += wsum[w];
        a.stats[(long long)row * a.slices + slice] = {bm, (float)s};
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

// Candidate c of a group as (order of its score, beam * vocab + token): c counts
// the rows' slices' keys; a row that is finished, or whose candidates are all
// -inf, offers its first tokens instead (and the finished one eos).
struct Cand {
    uint64_t score;
    uint64_t at;     // flat index, ~0: none
};

G4_DEV bool better(const Cand &x, const Cand &y) {
    return x.at != ~0ull && (y.at == ~0ull || x.score > y.score || (x.score == y.score && x.at < y.at));
}

__global__ void __launch_bounds__(kMergeThreads) k_beam_merge(BeamArgs a) {
    __shared__ double lse[kMaxBeams];       // of a live row
    __shared__ int kind[kMaxBeams];         // 0 live, 1 all -inf, 2 finished
    __shared__ uint64_t b_score[kMergeThreads / 32], b_at[kMergeThreads / 32];
    griddep_wait();
    const int grp = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int r = warp; r < a.beams; r += kMergeThreads / 32) {
        const SliceStat *st = a.stats + ((long long)grp * a.beams + r) * a.slices;
        float m = -INFINITY;
        for (int s = lane; s < a.slices; s += 32) m = fmaxf(m, st[s].max);
        m = warp_max(m);
        double sum = 0.0;
        for (int s = lane; s < a.slices; s += 32)
            if (st[s].max > -INFINITY) sum += (double)st[s].sum * exp((double)st[s].max - (double)m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            const float cum = a.scores[grp * a.beams + r];
            const bool done = a.finished && a.finished[grp * a.beams + r];
            kind[r] = cum - cum != 0.0f ? 1 : done ? 2 : m - m != 0.0f ? 1 : 0;
            lse[r] = kind[r] == 0 ? (double)m + log(sum) : 0.0;
        }
    }
    __syncthreads();
    const int per_row = a.slices * a.beams + 1;
    const int total = a.beams * per_row;
    Cand last = {~0ull, 0};
    for (int k = 0; k < a.beams; k++) {
        // best candidate after `last`
        Cand best = {0, ~0ull};
        for (int c = tid; c < total; c += kMergeThreads) {
            const int r = c / per_row, j = c % per_row;
            const float cum = a.scores[grp * a.beams + r];
            Cand x = {0, ~0ull};
            if (kind[r] == 0) {
                const uint64_t key = j < per_row - 1
                                         ? a.keys[((long long)grp * a.beams + r) * a.slices * a.beams + j] : 0;
                if (key) {
                    x.score = order_f64((double)cum + ((double)value_f32((uint32_t)(key >> 32)) - lse[r]));
                    x.at = (uint64_t)r * a.vocab + (uint32_t)~(uint32_t)key;
                }
            } else if (j < min(a.beams, a.vocab)) {
                x.score = order_f64(kind[r] == 2 && j == a.eos ? (double)cum : -(double)INFINITY);
                x.at = (uint64_t)r * a.vocab + j;
            } else if (j == per_row - 1 && kind[r] == 2 && a.eos >= min(a.beams, a.vocab)) {
                x.score = order_f64((double)cum);
                x.at = (uint64_t)r * a.vocab + a.eos;
            }
            if (x.at != ~0ull && (k == 0 || better(last, x)) && better(x, best)) best = x;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Cand y = {__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.at, o)};
            if (better(y, best)) best = y;
        }
        __syncthreads();
        if (lane == 0) { b_score[warp] = best.score; b_at[warp] = best.at; }
        __syncthreads();
        best = {b_score[0], b_at[0]};
        for (int w = 1; w < kMergeThreads / 32; w++) {
            const Cand y = {b_score[w], b_at[w]};
            if (better(y, best)) best = y;
        }
        last = best;
        if (tid == 0) {
            const int o = grp * a.beams + k;
            const int r = (int)(best.at / a.vocab), tok = (int)(best.at % a.vocab);
            a.out_scores[o] = (float)value_f64(best.score);
            a.parents[o] = r;
            a.tokens[o] = tok;
            if (a.out_finished)
                a.out_finished[o] = (a.finished && a.finished[grp * a.beams + r]) || tok == a.eos;
        }
    }
}

int slice_values(int) { return kThreads * 16; }

bool sizes_ok(int groups, int beams, int vocab) {
    return groups >= 0 && groups <= 65536 && beams >= 1 && beams <= kMaxBeams && vocab >= 1 && vocab <= 1 << 24;
}

template <typename T>
cudaError_t launch_rows(const BeamArgs &a, long long rows, cudaStream_t st) {
    const dim3 grid((unsigned)(rows * a.slices)), block(kThreads);
    const bool vec = ((uintptr_t)a.logits & 15) == 0 && a.stride * sizeof(T) % 16 == 0;
    return vec ? g4_launch(k_beam_rows<T, 16, true>, grid, block, 0, st, true, a)
               : g4_launch(k_beam_rows<T, 16, false>, grid, block, 0, st, true, a);
}

}  // namespace

extern "C" {

uint64_t g4_beam_workspace(int groups, int beams, int vocab) {
    if (!sizes_ok(groups, beams, vocab)) return 0;
    const uint64_t slices = (vocab + slice_values(0) - 1) / slice_values(0);
    return (uint64_t)(groups ? groups : 1) * beams * slices * (sizeof(SliceStat) + beams * sizeof(uint64_t));
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
    a.slice = slice_values(vocab);
    a.slices = (vocab + a.slice - 1) / a.slice;
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
