// g4_kv4.cu — the paged 4-bit KV cache: quantising writes, reads, and the pages
// of a beam search following its parents.
//
// All three move bytes and compute little: HBM bounds large calls, the launch
// and one memory round trip small ones. Measured: 34695 rows of 8 heads x 128 dimensions
// in bf16 written and read back 79 us (360 MB, 4.6 TB/s: finding a tile's rows and page is
// a chain of loads before each 16 tokens), 64 rows of 256 in fp32 6 us; reordering 16 x 8
// beams in 15 layers 15 us (64 MB, 4.3 TB/s), 4 beams in 12 layers 2.6 us.
#include <atomic>

#include <cuda_runtime.h>

#include "g4_kv4.cuh"

namespace {

constexpr int kThreads = 128;   // four warps, each its own 16 tokens x 64 dimensions
constexpr int kManyBlocks = 148 * 16;

// Tiles of 16 tokens: sequence b has the slots [offsets[b] / 16 + 2 b,
// offsets[b + 1] / 16 + 2 (b + 1)), at least as many as the records that its
// rows touch (q rows from any place in a record touch at most q / 16 + 2). So a
// grid of rows / 16 + 2 n covers every batch and no list is built. Finds the
// tile's rows: sequence, first row, rows, first position.
struct Tile {
    int seq, row, tokens;
    long long pos;
};

G4_DEV int slot_base(const Kv4View &c, int b) { return kv4_offset(c, b) / kKv4Rec + 2 * b; }

G4_DEV bool find_tile(const Kv4View &c, int slot, Tile &t) {
    int lo = 0, hi = c.n;                      // largest lo < n with slot_base(lo) <= slot
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (slot_base(c, mid) <= slot) lo = mid;
        else hi = mid;
    }
    const int r0 = kv4_offset(c, lo), r1 = kv4_offset(c, lo + 1);
    const long long p0 = c.start_pos[lo], p1 = p0 + (r1 - r0);
    const int k = slot - slot_base(c, lo);
    if (k < 0 || r1 <= r0) return false;
    // records of 16 positions, counted from the one that holds p0 (negative ones too)
    const long long first = (p0 >> 4) + k;
    const long long a = max(first * 16, p0), z = min(first * 16 + 16, p1);
    if (a >= z) return false;
    t.seq = lo;
    t.pos = a;
    t.row = r0 + (int)(a - p0);
    t.tokens = (int)(z - a);
    return true;
}

// Codes + 8 of 8 values of a group with scale s, a nibble each: x / s to the nearest
// integer, ties to even, exactly. x inv with one correction is x / s to within
// 2^-22 of half a step, which decides every case: where x / s is a tie it is one of
// fp32's values, and because (k + 1/2) s has 12 significant bits, any other x / s is
// more than 1.004 half steps away from a tie. (Bf16 inputs often meet ties, so that
// a division for those near one was taken by nearly every warp: 103 us for 32768
// rows of 8 x 128.) Adding 1.5 2^23 + 8 rounds to an integer, ties to even because
// the constant is even, whose low nibble is the code; the sum packs the nibbles.
G4_DEV uint32_t pack8(const float *x, float s, float inv) {
    constexpr float kMagic = 12582920.0f;                           // 0x4b400008
    const uint64_t inv2 = pk(inv, inv), minus_s = pk(-s, -s), one = pk(1.0f, 1.0f), magic = pk(kMagic, kMagic);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t v = pk(x[i], x[i + 1]), t = mul2(v, inv2);
        const float2 y = upk(fma2(fma2(fma2(t, minus_s, v), inv2, t), one, magic));
        w += __float_as_uint(y.x) << (4 * i);
        w += __float_as_uint(y.y) << (4 * i + 4);
    }
    constexpr uint32_t kTop = 0x4b400000u;                          // what each value adds above its nibble
    return w - (kTop + (kTop << 4) + (kTop << 8));                  // shifted by 12 and more it is 0 modulo 2^32
}

// Scale of a group from its largest absolute value (as bits, so that NaN and
// infinity are the largest) and its reciprocal to an ulp; inv 0: all codes are 0.
// The quotient by 7 is the correctly rounded one (a product and one correction), and
// rounding that to bf16 rounds the exact quotient: a bf16 tie times 7 has 12 bits.
G4_DEV uint32_t scale_of(uint32_t amax, float &s, float &inv) {
    constexpr float k7 = 0x1.24924ap-3f;                            // 1 / 7
    const float a = __uint_as_float(amax), q = a * k7;
    uint32_t b = __bfloat16_as_ushort(__float2bfloat16_rn(fmaf(fmaf(-7.0f, q, a), k7, q)));
    s = bf16_bits_f(b);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    if (amax - 0x0d800000u >= 0x7f000000u - 0x0d800000u) {          // < 2^-100, or >= 2^127, or not finite
        inv = 0.0f;
        b = amax >= 0x7f000000u ? 0x7fc0u : 0u;
    }
    return b;
}

// 8 values as they lie in memory, the largest |x| of them (as fp32 bits) and their
// values; those of 16 bits are compared two at a time.
template <typename T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
    G4_DEV void load(const T *p) {
        w[0] = reinterpret_cast<const uint4 *>(p)[0];
        if constexpr (sizeof(T) == 4) w[1] = reinterpret_cast<const uint4 *>(p)[1];
    }
    G4_DEV void zero() {
        w[0] = make_uint4(0, 0, 0, 0);
        if constexpr (sizeof(T) == 4) w[1] = make_uint4(0, 0, 0, 0);
    }
};
G4_DEV uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("max.u16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
G4_DEV uint32_t top(const Raw8<float> &r) {
    constexpr uint32_t A = 0x7fffffffu;
    return max(max(max(r.w[0].x & A, r.w[0].y & A), max(r.w[0].z & A, r.w[0].w & A)),
               max(max(r.w[1].x & A, r.w[1].y & A), max(r.w[1].z & A, r.w[1].w & A)));
}
template <typename T>
G4_DEV uint32_t top(const Raw8<T> &r) {
    const uint32_t m2 = max2(max2(r.w[0].x & 0x7fff7fffu, r.w[0].y & 0x7fff7fffu),
                             max2(r.w[0].z & 0x7fff7fffu, r.w[0].w & 0x7fff7fffu));
    const uint32_t m = max(m2 & 0xffffu, m2 >> 16);
    if constexpr (__is_same(T, __nv_bfloat16)) return m << 16;
    else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
}
G4_DEV void values(const Raw8<float> &r, float (&x)[8]) {
    const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __uint_as_float(w[i]);
}
template <typename T>
G4_DEV void values(const Raw8<T> &r, float (&x)[8]) {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (__is_same(T, __nv_bfloat16)) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}
template <typename T>
G4_DEV uint32_t codes(const Raw8<T> &r, float s, float inv) {
    float x[8];
    values(r, x);
    return inv == 0.0f ? 0x88888888u : pack8(x, s, inv);
}

// A warp takes units of a tile (kv head, group, K or V), `step` apart. Lane (g, t) =
// (lane / 4, lane % 4) holds what the attention kernel's lane will read: for K the 16
// dimensions 16 t of tokens g and g + 8, for V the 8 dimensions 8 g of tokens 2t,
// 2t+1, 2t+8, 2t+9. So a full tile's codes are one 512-byte store of the warp.
// (One unit per warp took 108 us for 32768 rows of 8 x 128 bf16: finding the tile
// and its page is two dependent loads, a unit's data one.)
// FULL: all 16 tokens of the record are rows.
template <typename T, bool FULL>
G4_DEV void write_units(const Kv4View &c, const T *k, long long k_stride, const T *v, long long v_stride,
                        uint8_t *rec0, long long row0, int t0, int t1, int unit, int step) {
    const int G = c.hd / kKv4Group, units = c.kv_heads * G * 2;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long long head_bytes = (long long)(17 * c.hd) << (c.page_shift - 4);
    const T *k0 = k + (row0 + g) * k_stride + 16 * t, *v0 = v + (row0 + 2 * t) * v_stride + 8 * g;
    auto in = [&](int tok) { return FULL || (tok >= t0 && tok < t1); };
    for (; unit < units; unit += step) {
        const int is_v = unit & 1, h = (unit >> 1) / G, grp = (unit >> 1) - h * G;
        uint8_t *rec = rec0 + h * head_bytes;
        uint16_t *ks = reinterpret_cast<uint16_t *>(rec + 16 * c.hd);
        const int at = h * c.hd + grp * kKv4Group;
        uint32_t w[4];
        if (!is_v) {
            Raw8<T> x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (in(g + 8 * (i >> 1))) x[i].load(k0 + at + (i >> 1) * 8 * k_stride + 8 * (i & 1));
                else x[i].zero();
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                uint32_t m = max(top(x[2 * i]), top(x[2 * i + 1]));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                float s, inv;
                const uint32_t b = scale_of(m, s, inv);
                w[2 * i] = codes(x[2 * i], s, inv);
                w[2 * i + 1] = codes(x[2 * i + 1], s, inv);
                const int tok = g + 8 * i;
                if (in(tok) && t == 0) ks[tok * G + grp] = (uint16_t)b;
                if (!FULL && in(tok))
                    *reinterpret_cast<uint2 *>(rec + grp * 512 + lane * 16 + 8 * i) =
                        make_uint2(w[2 * i], w[2 * i + 1]);
            }
            if (FULL) *reinterpret_cast<uint4 *>(rec + grp * 512 + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            Raw8<T> x[4];
            uint32_t m[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (in(2 * t + (j & 1) + 8 * (j >> 1))) x[j].load(v0 + at + ((j & 1) + 8 * (j >> 1)) * v_stride);
                else x[j].zero();
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                m[j] = top(x[j]);
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], o));
            }
            // lane (g, t) makes the scale of its token j = g % 4 and hands it round
            const uint32_t lo = g & 1 ? m[1] : m[0], hi = g & 1 ? m[3] : m[2];
            float s1, inv1;
            const uint32_t b = scale_of(g & 2 ? hi : lo, s1, inv1);
            uint8_t *to = rec + 8 * c.hd + grp * 512 + lane * 16;
            if (g < 4 && in(2 * t + (g & 1) + 8 * (g >> 1))) ks[16 * G + grp * 16 + t * 4 + g] = (uint16_t)b;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float s = __shfl_sync(0xffffffffu, s1, j * 4 + t), inv = __shfl_sync(0xffffffffu, inv1, j * 4 + t);
                w[j] = codes(x[j], s, inv);
                if (!FULL && in(2 * t + (j & 1) + 8 * (j >> 1))) *reinterpret_cast<uint32_t *>(to + 4 * j) = w[j];
            }
            if (FULL) *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 8) k_kv4_write(Kv4View c, const T *k, long long k_stride, const T *v,
                                                           long long v_stride, int parts) {
    griddep_wait();
    const int slot = blockIdx.x / parts, step = parts * (kThreads / 32);
    const int unit = (blockIdx.x - slot * parts) * (kThreads / 32) + (threadIdx.x >> 5);
    if (unit >= c.kv_heads * (c.hd / kKv4Group) * 2) return;
    Tile tile;
    if (!find_tile(c, slot, tile) || tile.pos < 0) return;
    uint8_t *rec0 = kv4_record(c, tile.seq, tile.pos, 0);
    if (!rec0) return;
    const int t0 = (int)(tile.pos & 15), t1 = t0 + tile.tokens;     // tokens of the record: [t0, t1)
    // first row of the record (may lie before the tensor; only rows of [t0, t1) are read)
    const long long row0 = (long long)tile.row - t0;
    if (tile.tokens == 16) write_units<T, true>(c, k, k_stride, v, v_stride, rec0, row0, t0, t1, unit, step);
    else write_units<T, false>(c, k, k_stride, v, v_stride, rec0, row0, t0, t1, unit, step);
}

G4_DEV void unpack8(uint32_t w, float s, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++)         // 2^23 + n, without a conversion
        x[i] = (__uint_as_float(0x4b000000u | ((w >> (4 * i)) & 15u)) - 8388616.0f) * s;
}

// The mirror of k_kv4_write. Rows at negative positions or without a page read as 0.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_kv4_read(Kv4View c, T *k, long long k_stride, T *v, long long v_stride,
                                                       int parts) {
    griddep_wait();
    const int slot = blockIdx.x / parts, step = parts * (kThreads / 32);
    const int G = c.hd / kKv4Group, units = c.kv_heads * G * 2;
    int unit = (blockIdx.x - slot * parts) * (kThreads / 32) + (threadIdx.x >> 5);
    if (unit >= units) return;
    Tile tile;
    if (!find_tile(c, slot, tile)) return;
    const uint8_t *rec0 = tile.pos < 0 ? nullptr : kv4_record(c, tile.seq, tile.pos, 0);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int t0 = (int)(tile.pos & 15), t1 = t0 + tile.tokens;
    const long long row0 = (long long)tile.row - t0;
    const long long head_bytes = (long long)(17 * c.hd) << (c.page_shift - 4);
    for (; unit < units; unit += step) {
        const int is_v = unit & 1, h = (unit >> 1) / G, grp = (unit >> 1) - h * G;
        uint4 q = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);   // codes of 0
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (rec0) {
            const uint8_t *rec = rec0 + h * head_bytes;
            const uint16_t *ks = reinterpret_cast<const uint16_t *>(rec + 16 * c.hd);
            q = *reinterpret_cast<const uint4 *>(rec + (is_v ? 8 * c.hd : 0) + grp * 512 + lane * 16);
            if (is_v) {
                const uint2 w = *reinterpret_cast<const uint2 *>(ks + 16 * G + grp * 16 + t * 4);
                s[0] = bf16_bits_f(w.x & 0xffffu);
                s[1] = bf16_bits_f(w.x >> 16);
                s[2] = bf16_bits_f(w.y & 0xffffu);
                s[3] = bf16_bits_f(w.y >> 16);
            } else {
                s[0] = bf16_bits_f(ks[g * G + grp]);
                s[1] = bf16_bits_f(ks[(g + 8) * G + grp]);
            }
        }
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        const long long at = (long long)h * c.hd + grp * kKv4Group;
        float x[8];
        if (!is_v) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int tok = g + 8 * i;
                if (tok < t0 || tok >= t1) continue;
                T *p = k + (row0 + tok) * k_stride + at + 16 * t;
                unpack8(w[2 * i], s[i], x);
                Kv4Vec<T>::store(p, x);
                unpack8(w[2 * i + 1], s[i], x);
                Kv4Vec<T>::store(p + 8, x);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int tok = 2 * t + (j & 1) + 8 * (j >> 1);
                if (tok < t0 || tok >= t1) continue;
                unpack8(w[j], s[j], x);
                Kv4Vec<T>::store(v + (row0 + tok) * v_stride + at + 8 * g, x);
            }
        }
    }
}

// ---- beams following their parents ------------------------------------------
constexpr int kMaxLayers = 64;
struct ReorderArgs {
    uint8_t *pages[kMaxLayers];
    int head_bytes[kMaxLayers];      // one page of one kv head
    int rec_bytes[kMaxLayers];
    int heads[kMaxLayers];
    int layers, num_pages, page_shift;
    int beams, table_stride;
    const int *parents, *lengths, *table_in, *spare_in;
    int *table_out, *spare_out;
};

// Grid (rows, layers + 1): block (i, l) copies beam i's part-full page in layer
// l, block (i, layers) writes its table row and spare page. Source pages are
// read only: a destination is a spare page, and no beam's table names one.
__global__ void __launch_bounds__(256) k_kv4_reorder(const __grid_constant__ ReorderArgs a) {
    griddep_wait();
    const int i = blockIdx.x, layer = blockIdx.y;
    const int grp = i / a.beams;
    int p = a.parents[i];
    p = (unsigned)p < (unsigned)a.beams ? grp * a.beams + p : i;
    const int len = max(a.lengths[grp], 0);
    const int full = len >> a.page_shift, left = len & ((1 << a.page_shift) - 1);
    const bool moved = p != i && left > 0 && full < a.table_stride;
    const int *mine = a.table_in + (long long)i * a.table_stride, *from = a.table_in + (long long)p * a.table_stride;
    const int src = moved ? from[full] : -1, dst = a.spare_in[i];
    const bool src_ok = (unsigned)src < (unsigned)a.num_pages, dst_ok = (unsigned)dst < (unsigned)a.num_pages;
    // A parent without a page there leaves nothing to copy: the spare page, whose old content
    // would become keys, stays a spare one and the beam has no page either.
    const bool none = moved && !src_ok && dst_ok;
    if (layer == a.layers) {
        int *out = a.table_out + (long long)i * a.table_stride;
        for (int j = threadIdx.x; j < a.table_stride; j += blockDim.x)
            out[j] = j < full ? from[j] : j == full && moved ? (none ? src : dst) : mine[j];
        if (threadIdx.x == 0) a.spare_out[i] = moved && !none ? mine[full] : dst;
        return;
    }
    if (!src_ok || !dst_ok || src == dst) return;
    const int hb = a.head_bytes[layer];
    const int n16 = ((left + kKv4Rec - 1) / kKv4Rec) * a.rec_bytes[layer] / 16;   // 16-byte pieces per head
    const uint8_t *s = a.pages[layer] + (long long)src * hb * a.heads[layer];
    uint8_t *d = a.pages[layer] + (long long)dst * hb * a.heads[layer];
    for (int h = 0; h < a.heads[layer]; h++, s += hb, d += hb) {
        const uint4 *s4 = reinterpret_cast<const uint4 *>(s);
        uint4 *d4 = reinterpret_cast<uint4 *>(d);
#pragma unroll 4
        for (int j = threadIdx.x; j < n16; j += 256) d4[j] = s4[j];
    }
}

std::atomic<int> g_starve{0};       // g4_test_kv4_attention_starve

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
bool aligned4(const void *p) { return ((uintptr_t)p & 3) == 0; }

template <typename T>
cudaError_t launch_move(bool write, const Kv4View &c, const void *k, long long ks, const void *v, long long vs,
                        cudaStream_t st) {
    // Blocks per tile: few tiles are spread over the GPU (64 rows: a unit per warp), many
    // keep their units together.
    const int units = c.kv_heads * (c.hd / kKv4Group) * 2, most = (units + kThreads / 32 - 1) / (kThreads / 32);
    const int slots = c.rows / kKv4Rec + 2 * c.n;
    const int parts = slots * most <= kManyBlocks ? most : (kManyBlocks + slots - 1) / slots;
    const unsigned blocks = (unsigned)slots * parts;
    if (write)
        return g4_launch(k_kv4_write<T>, dim3(blocks), dim3(kThreads), 0, st, true, c, (const T *)k, ks,
                         (const T *)v, vs, parts);
    return g4_launch(k_kv4_read<T>, dim3(blocks), dim3(kThreads), 0, st, true, c, (T *)k, ks, (T *)v, vs,
                     parts);
}

int move_rows(bool write, const g4_kv4_cache *cache, const g4_kv4_batch *batch, int type, const void *k,
              int64_t k_stride, const void *v, int64_t v_stride, void *stream) {
    Kv4View c;
    const int rc = kv4_view(cache, batch, &c);
    if (rc != G4_OK) return rc;
    if (!kv4_tensor_ok(k, k_stride, c.kv_heads, c.hd, type) || !kv4_tensor_ok(v, v_stride, c.kv_heads, c.hd, type))
        return G4_ERR_INVALID;
    if (c.n == 0 || c.rows == 0) return G4_OK;
    DeviceOf dev(c.pages);
    if (dev.status() != G4_OK) return dev.status();
    if (!dev.holds(k) || !dev.holds(v) || !dev.holds(c.offsets) || !dev.holds(c.start_pos) || !dev.holds(c.table))
        return G4_ERR_INVALID;
    cudaError_t e;
    if (type == G4_TYPE_F32) e = launch_move<float>(write, c, k, k_stride, v, v_stride, (cudaStream_t)stream);
    else if (type == G4_TYPE_BF16)
        e = launch_move<__nv_bfloat16>(write, c, k, k_stride, v, v_stride, (cudaStream_t)stream);
    else e = launch_move<__half>(write, c, k, k_stride, v, v_stride, (cudaStream_t)stream);
    return e == cudaSuccess ? G4_OK : G4_ERR_CUDA;
}

}  // namespace

size_t kv4_type_bytes(int type) { return type == G4_TYPE_F32 ? 4 : 2; }

DeviceOf::DeviceOf(const void *p) : status_(G4_ERR_CUDA) {
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return;
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) {
        status_ = G4_ERR_INVALID;
        return;
    }
    int cur = 0;
    if (cudaGetDevice(&cur) != cudaSuccess) return;
    dev_ = at.device;
    if (cur != dev_) {
        if (cudaSetDevice(dev_) != cudaSuccess) return;
        prev_ = cur;
    }
    status_ = G4_OK;
}
DeviceOf::~DeviceOf() {
    if (prev_ >= 0) cudaSetDevice(prev_);
}
bool DeviceOf::holds(const void *p) const {
    if (!p) return true;
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == dev_);
}

int kv4_check_cache(const g4_kv4_cache *c) {
    if (!c || !c->pages || !aligned16(c->pages) || c->num_pages < 1) return G4_ERR_INVALID;
    return g4_kv4_page_bytes(c->kv_heads, c->head_dim, c->page_size) ? G4_OK : G4_ERR_INVALID;
}

int kv4_view(const g4_kv4_cache *c, const g4_kv4_batch *b, Kv4View *v) {
    if (kv4_check_cache(c) != G4_OK || !b) return G4_ERR_INVALID;
    if (b->n < 0 || b->n > 65536 || b->rows < 0 || b->rows > 1 << 22 || b->table_stride < 1 ||
        (int64_t)b->table_stride * c->page_size > 1 << 30)
        return G4_ERR_INVALID;
    if (!b->offsets || !b->start_pos || !b->page_table || !aligned4(b->offsets) || !aligned4(b->start_pos) ||
        !aligned4(b->page_table))
        return G4_ERR_INVALID;
    v->pages = (uint8_t *)c->pages;
    v->page_bytes = (long long)g4_kv4_page_bytes(c->kv_heads, c->head_dim, c->page_size);
    v->num_pages = c->num_pages;
    v->page_shift = __builtin_ctz((unsigned)c->page_size);
    v->kv_heads = c->kv_heads;
    v->hd = c->head_dim;
    v->n = b->n;
    v->rows = b->rows;
    v->offsets = b->offsets;
    v->start_pos = b->start_pos;
    v->table = b->page_table;
    v->table_stride = b->table_stride;
    return G4_OK;
}

bool kv4_tensor_ok(const void *p, int64_t stride, int heads, int hd, int type) {
    if (type != G4_TYPE_F32 && type != G4_TYPE_BF16 && type != G4_TYPE_F16) return false;
    if (!p || !aligned16(p) || stride < (int64_t)heads * hd || stride > (int64_t)1 << 40) return false;
    return stride * (int64_t)kv4_type_bytes(type) % 16 == 0;
}

extern "C" {

uint64_t g4_kv4_page_bytes(int kv_heads, int head_dim, int page_size) {
    if (kv_heads < 1 || kv_heads > 256) return 0;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512) return 0;
    if (page_size < kKv4Rec || page_size > 1024 || (page_size & (page_size - 1))) return 0;
    return (uint64_t)kv_heads * (page_size / kKv4Rec) * 17 * head_dim;
}

int g4_kv4_write(const g4_kv4_cache *cache, const g4_kv4_batch *batch, int type, const void *k, int64_t k_stride,
                 const void *v, int64_t v_stride, void *stream) {
    return move_rows(true, cache, batch, type, k, k_stride, v, v_stride, stream);
}

int g4_kv4_read(const g4_kv4_cache *cache, const g4_kv4_batch *batch, int type, void *k, int64_t k_stride, void *v,
                int64_t v_stride, void *stream) {
    return move_rows(false, cache, batch, type, k, k_stride, v, v_stride, stream);
}

uint64_t g4_kv4_attention_workspace(const g4_kv4_cache *cache, const g4_kv4_batch *batch, int type, int q_heads) {
    Kv4View c;
    if (kv4_view(cache, batch, &c) != G4_OK) return 0;
    if (type != G4_TYPE_F32 && type != G4_TYPE_BF16 && type != G4_TYPE_F16) return 0;
    if (q_heads < c.kv_heads || q_heads % c.kv_heads || q_heads / c.kv_heads > 64) return 0;
    return g4_kv4_attention_ws(c, type, q_heads);
}

int g4_kv4_attention(const g4_kv4_cache *cache, const g4_kv4_batch *batch, int type, int q_heads, const void *q,
                     int64_t q_stride, void *out, int64_t out_stride, float scale, int window, void *workspace,
                     uint64_t workspace_bytes, void *stream) {
    const uint64_t need = g4_kv4_attention_workspace(cache, batch, type, q_heads);
    Kv4View c;
    if (!need || kv4_view(cache, batch, &c) != G4_OK) return G4_ERR_INVALID;
    if (!kv4_tensor_ok(q, q_stride, q_heads, c.hd, type) || !kv4_tensor_ok(out, out_stride, q_heads, c.hd, type))
        return G4_ERR_INVALID;
    if (!(scale == scale) || scale - scale != 0.0f || window < 0) return G4_ERR_INVALID;
    if (!workspace || !aligned16(workspace) || workspace_bytes < need) return G4_ERR_INVALID;
    if (c.n == 0 || c.rows == 0) return G4_OK;
    DeviceOf dev(c.pages);
    if (dev.status() != G4_OK) return dev.status();
    if (!dev.holds(q) || !dev.holds(out) || !dev.holds(c.offsets) || !dev.holds(c.start_pos) || !dev.holds(c.table) ||
        !dev.holds(workspace))
        return G4_ERR_INVALID;
    const cudaError_t e = g4_launch_kv4_attention(c, type, q_heads, q, q_stride, out, out_stride, scale, window,
                                                  workspace, g_starve.exchange(0), (cudaStream_t)stream);
    return e == cudaSuccess ? G4_OK : G4_ERR_CUDA;
}

int g4_test_kv4_attention_starve(int what) {
    if (what < 0 || what > 2) return G4_ERR_INVALID;
    g_starve = what;
    return G4_OK;
}

int g4_kv4_reorder(const g4_kv4_cache *caches, int layers, int groups, int beams, const int *parents,
                   const int *lengths, const int *table_in, int *table_out, int table_stride, const int *spare_in,
                   int *spare_out, void *stream) {
    if (!caches || layers < 1 || layers > kMaxLayers || groups < 0 || groups > 65536 || beams < 1 || beams > 32 ||
        table_stride < 1)
        return G4_ERR_INVALID;
    if (!parents || !lengths || !table_in || !table_out || !spare_in || !spare_out) return G4_ERR_INVALID;
    if (!aligned4(parents) || !aligned4(lengths) || !aligned4(table_in) || !aligned4(table_out) ||
        !aligned4(spare_in) || !aligned4(spare_out))
        return G4_ERR_INVALID;
    const long long rows = (long long)groups * beams;
    const size_t tb = (size_t)rows * table_stride * 4, sb = (size_t)rows * 4;
    const struct { const void *p; size_t n; } in[4] = {{table_in, tb}, {spare_in, sb}, {parents, sb}, {lengths, (size_t)groups * 4}};
    for (const auto &x : in)
        if (kv4_overlap(table_out, tb, x.p, x.n) || kv4_overlap(spare_out, sb, x.p, x.n)) return G4_ERR_INVALID;
    ReorderArgs a;
    for (int l = 0; l < layers; l++) {
        if (kv4_check_cache(&caches[l]) != G4_OK || caches[l].page_size != caches[0].page_size ||
            caches[l].num_pages != caches[0].num_pages)
            return G4_ERR_INVALID;
        a.pages[l] = (uint8_t *)caches[l].pages;
        a.rec_bytes[l] = 17 * caches[l].head_dim;
        a.head_bytes[l] = caches[l].page_size / kKv4Rec * a.rec_bytes[l];
        a.heads[l] = caches[l].kv_heads;
    }
    if (groups == 0) return G4_OK;
    DeviceOf dev(caches[0].pages);
    if (dev.status() != G4_OK) return dev.status();
    for (int l = 1; l < layers; l++)
        if (!dev.holds(caches[l].pages)) return G4_ERR_INVALID;
    if (!dev.holds(parents) || !dev.holds(lengths) || !dev.holds(table_in) || !dev.holds(table_out) ||
        !dev.holds(spare_in) || !dev.holds(spare_out))
        return G4_ERR_INVALID;
    a.layers = layers;
    a.num_pages = caches[0].num_pages;
    a.page_shift = __builtin_ctz((unsigned)caches[0].page_size);
    a.beams = beams;
    a.table_stride = table_stride;
    a.parents = parents;
    a.lengths = lengths;
    a.table_in = table_in;
    a.spare_in = spare_in;
    a.table_out = table_out;
    a.spare_out = spare_out;
    const cudaError_t e = g4_launch(k_kv4_reorder, dim3((unsigned)rows, layers + 1), dim3(256), 0,
                                    (cudaStream_t)stream, true, a);
    return e == cudaSuccess ? G4_OK : G4_ERR_CUDA;
}

}  // extern "C"
