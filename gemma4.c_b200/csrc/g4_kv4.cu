// g4_kv4.cu — the paged 4-bit KV cache: quantising writes, reads, and the pages
// of a beam search following its parents.
//
// All three move bytes and compute little: HBM bounds large calls, the launch
// and one memory round trip small ones.
#include <cuda_runtime.h>

#include "g4_kv4.cuh"

namespace {

constexpr int kThreads = 128;   // four warps, each its own 16 tokens x 64 dimensions

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

// Code + 8 of x for a group with scale s: x / s to the nearest integer, ties to
// even, exactly. x * inv is within 2^-21 of x / s (|x / s| < 8), so only values
// that close to a tie need the division, whose rounded quotient is a tie only
// if the exact one is: (k + 1/2) s has 12 significant bits, so any other x is
// further from it than half a step of the quotient.
G4_DEV uint32_t code_of(float x, float s, float inv) {
    const float t = x * inv;
    float r = rintf(t);
    if (fabsf(fabsf(t - r) - 0.5f) < 0x1p-18f) r = rintf(__fdiv_rn(x, s));
    return (uint32_t)(int)(fminf(fmaxf(r, -7.0f), 7.0f) + 8.0f);
}

// Scale of a group from its largest absolute value (as bits, so that NaN and
// infinity are the largest).
G4_DEV uint32_t scale_of(uint32_t amax, float &s, float &inv) {
    uint32_t b;
    if (amax >= 0x7f000000u) b = 0x7fc0u;                           // not finite, or >= 2^127
    else if (amax < 0x0d800000u) b = 0u;                            // < 2^-100
    else b = __bfloat16_as_ushort(__float2bfloat16_rn(__fdiv_rn(__uint_as_float(amax), 7.0f)));
    s = bf16_bits_f(b);
    inv = (b == 0u || b == 0x7fc0u) ? 0.0f : __frcp_rn(s);
    if (b == 0x7fc0u) s = 1.0f;
    return b;
}

template <int N>
G4_DEV uint32_t abs_max(const float (&x)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
}

G4_DEV uint32_t pack8(const float *x, float s, float inv, bool nan) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) w |= code_of(nan ? 0.0f : x[i], s, inv) << (4 * i);
    return w;
}

// One warp per (tile, kv head, K or V, group): lane (g, t) = (lane / 4, lane % 4)
// holds what the attention kernel's lane will read: for K the 16 dimensions 16 t
// of tokens g and g + 8, for V the 8 dimensions 8 g of tokens 2t, 2t+1, 2t+8,
// 2t+9. So a full tile's codes are one 512-byte store of the warp.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_kv4_write(Kv4View c, const T *k, long long k_stride, const T *v,
                                                        long long v_stride, int parts) {
    griddep_wait();
    const int slot = blockIdx.x / parts;
    const int unit = (blockIdx.x % parts) * (kThreads / 32) + (threadIdx.x >> 5);
    const int G = c.hd / kKv4Group;
    if (unit >= c.kv_heads * G * 2) return;
    Tile tile;
    if (!find_tile(c, slot, tile) || tile.pos < 0) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int is_v = unit & 1, grp = (unit >> 1) % G, h = (unit >> 1) / G;
    uint8_t *rec = kv4_record(c, tile.seq, tile.pos, h);
    if (!rec) return;
    const int t0 = (int)(tile.pos & 15), t1 = t0 + tile.tokens;     // tokens of the record: [t0, t1)
    // first row of the record (may lie before the tensor; only rows of [t0, t1) are read)
    const long long row0 = (long long)tile.row - t0;
    const bool full = tile.tokens == 16;
    uint16_t *ks = reinterpret_cast<uint16_t *>(rec + 16 * c.hd);
    if (!is_v) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int tok = g + 8 * i;
            const bool mine = tok >= t0 && tok < t1;
            float x[16];
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = 0.0f;
            if (mine) {
                const T *p = k + (row0 + tok) * k_stride + (long long)h * c.hd + grp * kKv4Group + 16 * t;
                float y[8];
                Kv4Vec<T>::load(p, y);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = y[j];
                Kv4Vec<T>::load(p + 8, y);
#pragma unroll
                for (int j = 0; j < 8; j++) x[8 + j] = y[j];
            }
            uint32_t m = abs_max(x);
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            float s, inv;
            const uint32_t b = scale_of(m, s, inv);
            w[2 * i] = pack8(x, s, inv, b == 0x7fc0u);
            w[2 * i + 1] = pack8(x + 8, s, inv, b == 0x7fc0u);
            if (mine && t == 0) ks[tok * G + grp] = (uint16_t)b;
            if (mine && !full)
                *reinterpret_cast<uint2 *>(rec + grp * 512 + lane * 16 + 8 * i) = make_uint2(w[2 * i], w[2 * i + 1]);
        }
        if (full) *reinterpret_cast<uint4 *>(rec + grp * 512 + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        uint32_t w[4];
        uint16_t *vs = ks + 16 * G + grp * 16 + t * 4;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int tok = 2 * t + (j & 1) + 8 * (j >> 1);
            const bool mine = tok >= t0 && tok < t1;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = 0.0f;
            if (mine) Kv4Vec<T>::load(v + (row0 + tok) * v_stride + (long long)h * c.hd + grp * kKv4Group + 8 * g, x);
            uint32_t m = abs_max(x);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            float s, inv;
            const uint32_t b = scale_of(m, s, inv);
            w[j] = pack8(x, s, inv, b == 0x7fc0u);
            if (mine && g == 0) vs[j] = (uint16_t)b;
            if (mine && !full)
                *reinterpret_cast<uint32_t *>(rec + 8 * c.hd + grp * 512 + lane * 16 + 4 * j) = w[j];
        }
        if (full)
            *reinterpret_cast<uint4 *>(rec + 8 * c.hd + grp * 512 + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

G4_DEV void unpack8(uint32_t w, float s, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)((int)((w >> (4 * i)) & 15u) - 8) * s;
}

// The mirror of k_kv4_write. Rows at negative positions or without a page read as 0.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_kv4_read(Kv4View c, T *k, long long k_stride, T *v, long long v_stride,
                                                       int parts) {
    griddep_wait();
    const int slot = blockIdx.x / parts;
    const int unit = (blockIdx.x % parts) * (kThreads / 32) + (threadIdx.x >> 5);
    const int G = c.hd / kKv4Group;
    if (unit >= c.kv_heads * G * 2) return;
    Tile tile;
    if (!find_tile(c, slot, tile)) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int is_v = unit & 1, grp = (unit >> 1) % G, h = (unit >> 1) / G;
    const uint8_t *rec = tile.pos < 0 ? nullptr : kv4_record(c, tile.seq, tile.pos, h);
    const int t0 = (int)(tile.pos & 15), t1 = t0 + tile.tokens;
    const long long row0 = (long long)tile.row - t0;
    const int code0 = is_v ? 8 * c.hd : 0;
    uint4 q = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);   // codes of 0
    if (rec) q = *reinterpret_cast<const uint4 *>(rec + code0 + grp * 512 + lane * 16);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    const uint16_t *ks = reinterpret_cast<const uint16_t *>(rec + 16 * c.hd);
    if (!is_v) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int tok = g + 8 * i;
            if (tok < t0 || tok >= t1) continue;
            const float s = rec ? bf16_bits_f(ks[tok * G + grp]) : 0.0f;
            T *p = k + (row0 + tok) * k_stride + (long long)h * c.hd + grp * kKv4Group + 16 * t;
            float x[8];
            unpack8(w[2 * i], s, x);
            Kv4Vec<T>::store(p, x);
            unpack8(w[2 * i + 1], s, x);
            Kv4Vec<T>::store(p + 8, x);
        }
    } else {
        const uint16_t *vs = ks + 16 * G + grp * 16 + t * 4;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int tok = 2 * t + (j & 1) + 8 * (j >> 1);
            if (tok < t0 || tok >= t1) continue;
            float x[8];
            unpack8(w[j], rec ? bf16_bits_f(vs[j]) : 0.0f, x);
            Kv4Vec<T>::store(v + (row0 + tok) * v_stride + (long long)h * c.hd + grp * kKv4Group + 8 * g, x);
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
    if (layer == a.layers) {
        int *out = a.table_out + (long long)i * a.table_stride;
        for (int j = threadIdx.x; j < a.table_stride; j += blockDim.x)
            out[j] = j < full ? from[j] : j == full && moved ? a.spare_in[i] : mine[j];
        if (threadIdx.x == 0) a.spare_out[i] = moved ? mine[full] : a.spare_in[i];
        return;
    }
    if (!moved) return;
    const int src = from[full], dst = a.spare_in[i];
    if ((unsigned)src >= (unsigned)a.num_pages || (unsigned)dst >= (unsigned)a.num_pages || src == dst) return;
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

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
bool aligned4(const void *p) { return ((uintptr_t)p & 3) == 0; }

template <typename T>
cudaError_t launch_move(bool write, const Kv4View &c, const void *k, long long ks, const void *v, long long vs,
                        cudaStream_t st) {
    const int units = c.kv_heads * (c.hd / kKv4Group) * 2;
    const int parts = (units + kThreads / 32 - 1) / (kThreads / 32);
    // rows <= 2^22, n <= 2^16 and parts <= 1024: below 2^31
    const unsigned blocks = (unsigned)((c.rows / kKv4Rec + 2 * c.n) * parts);
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
                                                  workspace, (cudaStream_t)stream);
    return e == cudaSuccess ? G4_OK : G4_ERR_CUDA;
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
    const uintptr_t tb = (uintptr_t)rows * table_stride * 4, sb = (uintptr_t)rows * 4;
    const uintptr_t ti = (uintptr_t)table_in, to = (uintptr_t)table_out, si = (uintptr_t)spare_in,
                    so = (uintptr_t)spare_out;
    if ((ti < to + tb && to < ti + tb) || (si < so + sb && so < si + sb)) return G4_ERR_INVALID;
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
