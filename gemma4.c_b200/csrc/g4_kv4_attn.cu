// g4_kv4_attn.cu — attention over the paged 4-bit KV cache.
#include <cuda_runtime.h>

#include "g4_kv4.cuh"

namespace {

G4_DEV void put(float *p, float x) { *p = x; }
G4_DEV void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
G4_DEV void put(__half *p, float x) { *p = __float2half_rn(x); }

// One CTA per (token row, query head), one warp per key, online softmax per warp.
template <int HD, typename T>
__global__ void __launch_bounds__(128) k_kv4_attn_row(Kv4View c, int q_heads, const T *q, long long q_stride, T *out,
                                                      long long out_stride, float scale, int window) {
    constexpr int D = HD / 32, G = HD / kKv4Group;
    __shared__ float so[4][HD], sm[4], sl[4];
    const int row = blockIdx.x / q_heads, head = blockIdx.x % q_heads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int lo = 0, hi = c.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (kv4_offset(c, mid) <= row) lo = mid;
        else hi = mid;
    }
    // empty sequences share an offset with the next one: the last of them was found
    if (row < kv4_offset(c, lo) || row >= kv4_offset(c, lo + 1)) return;
    const long long pos = (long long)c.start_pos[lo] + row - kv4_offset(c, lo);
    const long long first = window ? max(pos - window + 1, 0ll) : 0;
    const long long last = min(pos, ((long long)c.table_stride << c.page_shift) - 1);
    const int h = head / (q_heads / c.kv_heads);
    float qv[D], o[D], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < D; i++) {
        qv[i] = (float)q[row * q_stride + (long long)head * HD + lane + 32 * i];
        o[i] = 0.0f;
    }
    for (long long j = first + warp; j <= last; j += 4) {
        const uint8_t *rec = kv4_record(c, lo, j, h);
        if (!rec) continue;
        const int t = (int)(j & 15);
        const uint16_t *ks = reinterpret_cast<const uint16_t *>(rec + 16 * HD), *vs = ks + 16 * G;
        float s = 0.0f, v[D];
#pragma unroll
        for (int i = 0; i < D; i++) {
            const int d = lane + 32 * i, grp = d >> 6, e = d & 63, sh = (d & 1) * 4;
            const int kb = grp * 512 + (t & 7) * 64 + (e >> 4) * 16 + (t >> 3) * 8 + ((e & 15) >> 1);
            const int vb = 8 * HD + grp * 512 + (e >> 3) * 64 + (t >> 1 & 3) * 16 + (t >> 3) * 8 + (t & 1) * 4 +
                           ((e & 7) >> 1);
            s += qv[i] * ((float)((rec[kb] >> sh & 15) - 8) * bf16_bits_f(ks[t * G + grp]));
            v[i] = (float)((rec[vb] >> sh & 15) - 8) *
                   bf16_bits_f(vs[grp * 16 + (t >> 1 & 3) * 4 + (t >> 3) * 2 + (t & 1)]);
        }
        s = warp_sum(s) * scale;
        const float mn = fmaxf(m, s), a = expf(m - mn), p = expf(s - mn);
        l = l * a + p;
#pragma unroll
        for (int i = 0; i < D; i++) o[i] = o[i] * a + p * v[i];
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < D; i++) so[warp][lane + 32 * i] = o[i];
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
    __syncthreads();
    const float mt = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float a[4], lt = 0.0f;
    for (int w = 0; w < 4; w++) {
        a[w] = mt == -INFINITY ? 0.0f : expf(sm[w] - mt);
        lt += a[w] * sl[w];
    }
    const bool empty = mt == -INFINITY && lt == 0.0f;
    for (int d = threadIdx.x; d < HD; d += 128) {
        float x = 0.0f;
        for (int w = 0; w < 4; w++) x += a[w] * so[w][d];
        put(out + row * out_stride + (long long)head * HD + d, empty ? 0.0f : x / lt);
    }
}

template <int HD>
cudaError_t launch_row(const Kv4View &c, int type, int q_heads, const void *q, long long qs, void *out, long long os,
                       float scale, int window, cudaStream_t st) {
    const dim3 grid((unsigned)c.rows * q_heads), block(128);
    if (type == G4_TYPE_F32)
        return g4_launch(k_kv4_attn_row<HD, float>, grid, block, 0, st, false, c, q_heads, (const float *)q, qs,
                         (float *)out, os, scale, window);
    if (type == G4_TYPE_BF16)
        return g4_launch(k_kv4_attn_row<HD, __nv_bfloat16>, grid, block, 0, st, false, c, q_heads,
                         (const __nv_bfloat16 *)q, qs, (__nv_bfloat16 *)out, os, scale, window);
    return g4_launch(k_kv4_attn_row<HD, __half>, grid, block, 0, st, false, c, q_heads, (const __half *)q, qs,
                     (__half *)out, os, scale, window);
}

}  // namespace

size_t g4_kv4_attention_ws(const Kv4View &, int, int) { return 16; }

cudaError_t g4_launch_kv4_attention(const Kv4View &c, int type, int q_heads, const void *q, long long q_stride,
                                    void *out, long long out_stride, float scale, int window, void *,
                                    cudaStream_t st) {
    if (c.hd == 64) return launch_row<64>(c, type, q_heads, q, q_stride, out, out_stride, scale, window, st);
    if (c.hd == 128) return launch_row<128>(c, type, q_heads, q, q_stride, out, out_stride, scale, window, st);
    if (c.hd == 256) return launch_row<256>(c, type, q_heads, q, q_stride, out, out_stride, scale, window, st);
    return launch_row<512>(c, type, q_heads, q, q_stride, out, out_stride, scale, window, st);
}
