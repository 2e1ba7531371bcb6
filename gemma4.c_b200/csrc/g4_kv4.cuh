// g4_kv4.cuh — the paged 4-bit KV cache (include/g4cuda.h): what its kernels
// share. A record is 16 tokens of one kv head: 17 * hd bytes, codes in the order
// in which the warps of the attention kernel read them as tensor-core operands.
#pragma once
#include <cuda_bf16.h>

#include "../../include/g4cuda.h"
#include "g4_common.cuh"
#include "g4_internal.h"

constexpr int kKv4Rec = 16;               // tokens per record
constexpr int kKv4Group = 64;             // dimensions per scale

// A batch and its cache as the kernels take them.
struct Kv4View {
    uint8_t *pages;
    long long page_bytes;
    int num_pages, page_shift;
    int kv_heads, hd;
    int n, rows;
    const int *offsets, *start_pos, *table;
    int table_stride;
};

G4_DEV int kv4_rec_bytes(int hd) { return 17 * hd; }

// offsets[i], inside the tensors whatever the array holds
G4_DEV int kv4_offset(const Kv4View &c, int i) { return min(max(c.offsets[i], 0), c.rows); }

// Record of 16 tokens that holds position `pos` (>= 0) of sequence `seq` for kv
// head `h`, NULL where the sequence has no page.
G4_DEV uint8_t *kv4_record(const Kv4View &c, int seq, long long pos, int h) {
    const long long slot = pos >> c.page_shift;
    if (slot >= c.table_stride) return nullptr;
    const int page = c.table[(long long)seq * c.table_stride + slot];
    if ((unsigned)page >= (unsigned)c.num_pages) return nullptr;
    const int rec = (int)(pos & ((1 << c.page_shift) - 1)) / kKv4Rec;
    return c.pages + page * c.page_bytes + (long long)((h << c.page_shift) / kKv4Rec + rec) * kv4_rec_bytes(c.hd);
}

G4_DEV float bf16_bits_f(uint32_t b) { return __uint_as_float(b << 16); }

// ---- values of the three tensor types -------------------------------------
template <typename T>
struct Kv4Vec;   // 8 consecutive values, 16-byte aligned
template <>
struct Kv4Vec<float> {
    static G4_DEV void load(const float *p, float (&x)[8]) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    static G4_DEV void store(float *p, const float (&x)[8]) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
};
template <>
struct Kv4Vec<__nv_bfloat16> {
    static G4_DEV void load(const __nv_bfloat16 *p, float (&x)[8]) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static G4_DEV void store(__nv_bfloat16 *p, const float (&x)[8]) {
        __nv_bfloat162 h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(h);
    }
};
template <>
struct Kv4Vec<__half> {
    static G4_DEV void load(const __half *p, float (&x)[8]) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        const __half2 *h = reinterpret_cast<const __half2 *>(&a);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
    static G4_DEV void store(__half *p, const float (&x)[8]) {
        __half2 h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(h);
    }
};

// ---- host side --------------------------------------------------------------
// Argument checks and the view; G4_ERR_INVALID for what the kernels do not take.
int kv4_check_cache(const g4_kv4_cache *c);
int kv4_view(const g4_kv4_cache *c, const g4_kv4_batch *b, Kv4View *v);
// type is known and rows of `heads` heads start every `stride` elements, 16-byte aligned
bool kv4_tensor_ok(const void *p, int64_t stride, int heads, int hd, int type);
size_t kv4_type_bytes(int type);
// whether [a, a + an) and [b, b + bn) have a byte in common
inline bool kv4_overlap(const void *a, size_t an, const void *b, size_t bn) {
    return a && b && an && bn && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}

// Makes the device that holds `p` current for a scope; ok() is false when one
// of the pointers is not device memory of that device.
class DeviceOf {
  public:
    explicit DeviceOf(const void *p);
    ~DeviceOf();
    DeviceOf(const DeviceOf &) = delete;
    bool holds(const void *p) const;   // NULL counts as held
    int status() const { return status_; }

  private:
    int dev_ = -1, prev_ = -1, status_;
};

cudaError_t g4_launch_kv4_attention(const Kv4View &c, int type, int q_heads, const void *q, long long q_stride,
                                    void *out, long long out_stride, float scale, int window, void *ws, int starve,
                                    cudaStream_t st);      // starve: g4_test_kv4_attention_starve
size_t g4_kv4_attention_ws(const Kv4View &c, int type, int q_heads);
// Many query rows per sequence and kv head go to the tcgen05 tiles of 128 rows, few to
// tiles of 8 (g4_kv4_attn.cu), whose time grows with the rows while the other's starts at 33
// (256 dimensions) to 43 us (512) for a context of 4000. Measured on either side, us of the small
// and the large tiles: 16 sequences, 512 dimensions, 8 tokens x 8 heads on average 71 / 120, 16 tokens
// 127 / 124, 33 tokens 236 / 176; 256 dimensions, 16 tokens 74 / 69; 128 dimensions, 8 kv heads
// of 4, 16 tokens 134 / 169, 33 tokens 250 / 205. Fewer than four sequences and heads of many
// dimensions leave the large tiles less to share out: one sequence and kv head of 512
// dimensions, 64 tokens x 8 heads 47 / 50, 128 tokens 80 / 53; of 256 dimensions 35 / 37 and
// 51 / 36. Hence their own bound.
constexpr int kManyRows = 112, kManyRowsAlone = 576;
inline bool many_rows(const Kv4View &c, int q_heads) {
    const long long from = c.hd >= 256 && (long long)c.n * c.kv_heads < 4 ? kManyRowsAlone : kManyRows;
    return (long long)c.rows * (q_heads / c.kv_heads) >= from * c.n;
}
// g4_kv4_prompt.cu: the same for many query rows per sequence
size_t kv4_prompt_ws(const Kv4View &c, int type, int q_heads);
cudaError_t kv4_launch_prompt(const Kv4View &c, int type, int q_heads, const void *q, long long q_stride, void *out,
                              long long out_stride, float scale, int window, void *ws, int starve, cudaStream_t st);
