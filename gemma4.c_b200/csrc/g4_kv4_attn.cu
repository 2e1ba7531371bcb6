// g4_kv4_attn.cu — attention over the paged 4-bit KV cache.
//
// out = softmax(scale q K^T) V per token row and query head; K and V are codes
// c in -7..7 times a scale per token and group of 64 dimensions:
//   s_j = sum_G ks_jG (q_G . c_jG),   o_G = sum_j (p_j vs_jG) c_jG
// so both products run on the codes themselves and the scales are applied to
// scores and probabilities.
//
// One token of one sequence reads each cached byte once for all the query heads
// of its kv head, so HBM bounds it; per byte the tensor cores do little and the
// conversion of codes to operands is what has to be cheap. Hence mma.sync (the
// operands come straight from registers; a tcgen05 tile would need the converted
// codes written to shared memory again, and 8 heads use 1/16 of its rows) with
// the keys as M and 8 query rows as N (m16n8k16), and the cache laid out so that
// a lane's 16 bytes of a record are exactly its operands:
//   S^T = K Q^T  fp16. A nibble n = c + 8 in the low bits of an fp16 is the
//                subnormal n 2^-24 (16 n 2^-24 one nibble up): one AND makes two
//                operands. The 8 is taken off in the accumulator's start value,
//                -8 sum(q), whose truncation is the same for every key (codes without
//                the 8: outputs 4.8e-6 off, with it 2.4e-6). q is scaled per row to
//                2^13..2^14 and, if fp32, split into high and low halves (22 bits),
//                each with an accumulator of its own: the tensor core truncates by the
//                size of the sum (in one: 3.5e-6; 1 % of a 64-sequence step).
//   O^T = V^T P^T  bf16, whose range needs no common factor over the scales. A
//                nibble is the bf16 subnormal n 2^-133 (16 n 2^-133 one nibble up);
//                a packed add takes the 8 off, because the accumulator runs over all
//                keys and an offset there would add up the truncations of the tensor
//                core. p is 2^80 times too large to keep sums away from 2^-126: values
//                up to 2^38 times a code are safe. p vs is split into high and low
//                bf16: for fp32 outputs from the fp32 product (2^-18 of it is lost, a
//                third of what they are off; a third term would take 5 % longer), for
//                others by packed FMAs on p's own halves (16 bits).
// Every warp streams its own records of 16 keys through a ring in shared memory
// and keeps its own running maximum, sum and output; the warps meet once per
// sequence and head. Work is counted in records over all (sequence, row tile, kv
// head) and cut into one even run per CTA, so ragged batches and one long
// sequence fill the GPU alike; a sequence cut between CTAs leaves partial
// results that a second kernel joins in order.
//
// Measured (GPU time, both kernels): 64 sequences of 128 to 8704 tokens, one kv head of
// 512 dimensions, 8 fp32 query heads each 36 us (79 MB of records, 12.1 us at HBM's
// rate); one sequence of 131072 tokens 34 us (10.9); 32 sequences up to 16384, 8 kv heads
// of 128 dimensions, 32 bf16 heads 39 us (12.1); a window of 512 tokens 13 us. An SM
// takes about 570 clocks for a record of 512 dimensions where its share of HBM delivers
// one in 378. The tensor pipe is 30 % busy and 39 % of the issue slots are used, so it is
// latency: two warps a scheduler (255 registers), the dependent MMAs of a group's score, then
// maximum, exponentials and P V. Not better: two warps a record, Q K of the next record beside P V.
#include <algorithm>

#include <cuda_runtime.h>

#include "g4_kv4.cuh"

namespace {

constexpr int kRows = 8;          // query rows of a tile (tokens x heads of one kv head)
constexpr int kStreams = 8;       // warps of a CTA, each with a record of its own
constexpr int kThreads = kStreams * 32;
constexpr int kSms = 148;
constexpr int kJoinThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;                      // log2 of how far p may pass 1
constexpr float kUp = 0x1p80f;                      // p is 2^80 times too large
constexpr float kEven = 0x1p53f, kOdd = 0x1p49f;    // outputs: 2^133 / 2^80, 16 times less for odd dimensions

template <int HD>
struct Cfg {
    static constexpr int G = HD / kKv4Group;
    static constexpr int kRec = 17 * HD;
    static constexpr int kStages = HD >= 256 ? 3 : HD == 128 ? 4 : 6;
    static constexpr int kOcc = HD == 512 ? 1 : 2;
    static constexpr int kCtas = kSms * kOcc;
    static constexpr int kWhole = HD >= 256 ? 40 : 64;          // records of an item that is not cut
    static constexpr int kRing = kStreams * kStages * kRec;
    static constexpr int kQ = G * 1024;                         // operands of the query tile (one half)
    static constexpr int kPad = HD + 2;                        // row of a warp's output when the warps meet
    static constexpr int kSlot = kRows * HD;                    // floats of one partial output
    static_assert(kStages * kRec >= kRows * kPad * 4, "a stream's ring holds its output tile");
};

struct AttnP {
    Kv4View c;
    int type;
    unsigned group;               // query heads per kv head
    const void *q;
    void *out;
    long long q_stride, out_stride;
    float scale;
    int window;
    int whole;                    // items are not cut: there is nothing to join
    float *slots;                 // partial outputs [2 per CTA][8][HD]
    float *stats;                 // their maxima and sums [2 per CTA][2][8]
};

G4_DEV void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
G4_DEV void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

G4_DEV void mma_h(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
G4_DEV void mma_b(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
G4_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 8x8 matrix of 16-bit values across the warp: (row lane / 4, columns 2 (lane % 4), + 1) transposed
G4_DEV uint32_t movm(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// fp32 a (row g, column 2t), b (row g, column 2t + 1) of an 8x8 block -> (row 2t, column g), (row 2t + 1, column g)
G4_DEV void transpose2(float &a, float &b) {
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    const uint32_t lo = movm(__byte_perm(x, y, 0x5410)), hi = movm(__byte_perm(x, y, 0x7632));
    a = __uint_as_float(__byte_perm(lo, hi, 0x5410));
    b = __uint_as_float(__byte_perm(lo, hi, 0x7632));
}
G4_DEV uint32_t add_b(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
G4_DEV uint32_t mul_b(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
G4_DEV uint32_t fma_b(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t y;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(a), "r"(b), "r"(c));
    return y;
}
// Codes of the low nibble of each half's low byte as bf16 c 2^-133, of the high nibble as 16 c 2^-133
G4_DEV uint32_t code_lo(uint32_t x) { return add_b(x & 0x000f000fu, 0x80088008u); }
G4_DEV uint32_t code_hi(uint32_t x) { return add_b(x & 0x00f000f0u, 0x80808080u); }
G4_DEV uint32_t pack_b(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
G4_DEV uint32_t pack_h(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
G4_DEV float2 unpack_h(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }

G4_DEV void load8(const void *p, int type, long long i, float (&x)[8]) {
    if (type == G4_TYPE_F32) Kv4Vec<float>::load((const float *)p + i, x);
    else if (type == G4_TYPE_BF16) Kv4Vec<__nv_bfloat16>::load((const __nv_bfloat16 *)p + i, x);
    else Kv4Vec<__half>::load((const __half *)p + i, x);
}
G4_DEV void store8(void *p, int type, long long i, const float (&x)[8]) {
    if (type == G4_TYPE_F32) Kv4Vec<float>::store((float *)p + i, x);
    else if (type == G4_TYPE_BF16) Kv4Vec<__nv_bfloat16>::store((__nv_bfloat16 *)p + i, x);
    else Kv4Vec<__half>::store((__half *)p + i, x);
}

G4_DEV void store2(void *p, int type, long long i, float x, float y) {
    if (type == G4_TYPE_F32) *reinterpret_cast<float2 *>((float *)p + i) = make_float2(x, y);
    else *reinterpret_cast<uint32_t *>((uint16_t *)p + i) = type == G4_TYPE_BF16 ? pack_b(x, y) : pack_h(x, y);
}

// N bf16 scales, and one of a pair as fp32
template <int N>
G4_DEV void load_scales(const void *p, uint32_t (&w)[(N + 1) / 2]) {
    static_assert(N == 8 || N == 4 || N == 2 || N == 1, "the groups of a head");
    if constexpr (N == 8) {
        const uint4 x = *reinterpret_cast<const uint4 *>(p);
        w[0] = x.x;
        w[1] = x.y;
        w[2] = x.z;
        w[3] = x.w;
    } else if constexpr (N == 4) {
        const uint2 x = *reinterpret_cast<const uint2 *>(p);
        w[0] = x.x;
        w[1] = x.y;
    } else if constexpr (N == 2) w[0] = *reinterpret_cast<const uint32_t *>(p);
    else w[0] = *reinterpret_cast<const uint16_t *>(p);
}
G4_DEV float half_of(uint32_t w, int i) { return __uint_as_float(i ? w & 0xffff0000u : w << 16); }

// p times two bf16 scales as high and low bf16: 2^-18 of the product is lost
G4_DEV void split(uint64_t p, uint32_t vs, uint32_t &h, uint32_t &l) {
    const float2 x = upk(mul2(p, pk(half_of(vs, 0), half_of(vs, 1))));
    h = pack_b(x.x, x.y);
    l = pack_b(x.x - half_of(h, 0), x.y - half_of(h, 1));
}

constexpr int kItemCost = 16;
constexpr int kSeqs = 32;         // sequences described in shared memory at a time

// ---- the schedule -------------------------------------------------------------
// Sequence b: its rows in tiles of kRows, each tile x kv head an item of `recs`
// records (those that the sequence's rows see between them; a tile skips what
// its own rows do not see; at least 1, so that empty rows are written). An item
// counts kItemCost + recs units of work: its queries, the meeting of its warps and
// its output take about as long as kItemCost records (a 64-sequence step with
// contexts of 128 to 8704: the CTAs that got only short sequences took 60 us, the
// others 28, when items counted their records alone).
struct Seq {
    int row0, q, tiles, recs, rec0;
    long long pos0;
};

G4_DEV Seq seq_of(const AttnP &p, int b) {
    Seq s;
    s.row0 = kv4_offset(p.c, b);
    s.q = max(kv4_offset(p.c, b + 1) - s.row0, 0);
    s.pos0 = p.c.start_pos[b];
    s.tiles = (s.q * p.group + kRows - 1) / kRows;            // q <= 2^22, group <= 64
    const long long lo = p.window ? max(s.pos0 - p.window + 1, 0ll) : 0;
    const long long hi = min(s.pos0 + s.q - 1, ((long long)p.c.table_stride << p.c.page_shift) - 1);
    s.rec0 = (int)(lo >> 4);
    s.recs = hi < lo ? 1 : (int)((hi >> 4) - (lo >> 4)) + 1;
    return s;
}
G4_DEV long long work_of(const AttnP &p, const Seq &s) {
    return (long long)s.tiles * p.c.kv_heads * (s.recs + kItemCost);
}

// Total work, and the sequence in which unit `w` of it lies with w's offset in
// that sequence's work. Every thread of a block of N calls them.
template <int N>
struct Scan {
    long long warp[N / 32], off;
    int seq;
};
template <int N>
G4_DEV long long scan_total(const AttnP &p, Scan<N> &s, int per, long long &before, long long &mine) {
    const int tid = threadIdx.x, lane = tid & 31;
    mine = 0;
    // (bounded so that the sums stay in range for offsets that are not ascending as well)
    for (int b = tid * per; b < min((tid + 1) * per, p.c.n); b++) mine = min(mine + work_of(p, seq_of(p, b)), 1ll << 50);
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) s.warp[tid >> 5] = inc;
    __syncthreads();
    long long total = 0, base = 0;
#pragma unroll
    for (int i = 0; i < N / 32; i++) {
        if (i < (tid >> 5)) base += s.warp[i];
        total += s.warp[i];
    }
    before = base + inc - mine;
    return total;
}
template <int N>
G4_DEV void find_work(const AttnP &p, Scan<N> &s, int per, long long before, long long mine, long long w) {
    if (w >= before && w < before + mine) {
        long long at = before;
        int b = threadIdx.x * per;
        for (;; b++) {
            const long long x = work_of(p, seq_of(p, b));
            if (w < at + x) break;
            at += x;
        }
        s.seq = b;
        s.off = w - at;
    }
    __syncthreads();
}
G4_DEV long long share_of(long long total, int ctas) {
    // a 64-bit division costs as much as a load; most totals fit 32 bits
    const unsigned long long t = (unsigned long long)total + ctas - 1;
    const long long s = t >> 32 ? (long long)(t / ctas) : (long long)((unsigned)t / (unsigned)ctas);
    return max(s, (long long)kItemCost + kStreams);      // at least a round of records for who starts an item
}
// x / y and x % y for 0 <= x, 0 < y < 2^31
G4_DEV void divide(long long x, int y, int &q, int &r) {
    if ((unsigned long long)x >> 32) {
        q = (int)(x / y);
        r = (int)(x - (long long)q * y);
    } else {
        q = (int)((unsigned)x / (unsigned)y);
        r = (int)((unsigned)x - (unsigned)q * (unsigned)y);
    }
}

// ---- the streaming kernel -------------------------------------------------------
// What a CTA does of one item: records [ra, rb) of sequence b for kv head h and
// the rows [tile * kRows, + valid) of its group.
struct Item {
    int b, h, tile, valid, row0;
    int ra, rb;
    int all0, all1;            // every row sees the keys all0..all1
    long long pos0;
    int whole, starts, none;   // none: the CTA has no more work
};

// The CTA's way through its work, kept in shared memory by its last warp: the
// sequence (a run of kSeqs of them described at a time), the item of it and the
// unit of that where the next item starts.
struct Walk {
    long long left;
    int b, cached, item, unit;
    Seq seqs[kSeqs];
};

// The next item, by one whole warp.
G4_DEV void next_item(const AttnP &p, Walk &w, Item &out) {
    const int lane = threadIdx.x & 31, kvh = p.c.kv_heads;
    if (w.left <= 0) {
        if (lane == 0) out.none = 1;
        return;
    }
    int b = w.b, item = w.item;
    for (;; b++, item = 0) {
        if (b >= w.cached + kSeqs) {
            __syncwarp();
            if (b + lane < p.c.n) w.seqs[lane] = seq_of(p, b + lane);
            if (lane == 0) w.cached = b;
            __syncwarp();
        }
        if (item < w.seqs[b - w.cached].tiles * kvh) break;         // an empty sequence has no items
    }
    __syncwarp();
    if (lane) return;
    const int cap = p.c.table_stride << p.c.page_shift;              // <= 2^30
    const Seq s = w.seqs[b - w.cached];
    // units [u0, u1) of the item, of which the first kItemCost are no records: who
    // holds only such leaves the item to the next CTA
    const int size = s.recs + kItemCost, u0 = w.unit, u1 = p.whole ? size : (int)min((long long)size, u0 + w.left);
    const int r0 = max(u0 - kItemCost, 0), r1 = u1 - kItemCost;
    w.left -= u1 - u0;
    w.b = b;
    w.item = item + 1;
    w.unit = 0;
    if (r1 <= 0) {             // only at the end of the CTA's work; nothing else of `out` is set
        out.none = 1;
        return;
    }
    Item it;
    it.none = 0;
    it.b = b;
    it.tile = (unsigned)item / (unsigned)kvh;
    it.h = item - it.tile * kvh;
    it.whole = r0 == 0 && r1 == s.recs;
    it.starts = r0 == 0;
    it.row0 = s.row0;
    it.pos0 = s.pos0;
    // rows are (token, head of the group), token-major
    const unsigned first = it.tile * kRows;
    it.valid = min((int)(s.q * p.group - first), kRows);
    const long long pos_first = s.pos0 + first / p.group, pos_last = s.pos0 + (first + it.valid - 1) / p.group;
    const int see0 = p.window ? (int)min(max(pos_first - p.window + 1, 0ll), (long long)cap) : 0;
    const int see1 = (int)max(min(pos_last, (long long)cap - 1), -1ll);              // some row sees [see0, see1]
    it.all0 = p.window ? (int)min(max(pos_last - p.window + 1, 0ll), (long long)cap) : 0;
    it.all1 = (int)max(min(pos_first, (long long)cap - 1), -1ll);
    it.ra = max(s.rec0 + r0, see0 >> 4);
    it.rb = see1 < see0 ? it.ra : min(s.rec0 + r1, (see1 >> 4) + 1);
    out = it;
}

// STARVE: the test aid g4_test_kv4_attention_starve.
template <int HD, bool HILO, bool STARVE>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::kOcc) k_kv4_attn(const __grid_constant__ AttnP p) {
    using C = Cfg<HD>;
    constexpr int G = C::G, REC = C::kRec, ST = C::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;
    uint4 *qhi = reinterpret_cast<uint4 *>(smem + C::kRing);            // [HD / 64][2][32] (lane's operands of two steps)
    uint4 *qlo = qhi + C::kQ / 16;
    float *qoff = reinterpret_cast<float *>(smem + C::kRing + (HILO ? 2 : 1) * C::kQ);   // [HD / 64][8]: -8 sum q
    __shared__ Scan<kThreads> scan;
    __shared__ Walk walk;
    __shared__ Item items[2];
    __shared__ float row_scale[kRows], row_max[2][kStreams], sm_m[kStreams][kRows], sm_l[kStreams][kRows];
    __shared__ uint64_t full[kStreams][ST];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int stream = warp;
    const unsigned group = p.group;

    if (tid < kStreams * ST) mbar_init(&full[0][0] + tid, 1);
    mbar_fence_init();
    griddep_wait();
    const int per = (p.c.n + kThreads - 1) / kThreads;
    long long before, mine;
    const long long total = scan_total(p, scan, per, before, mine);
    const long long share = share_of(total, C::kCtas);
    const long long w0 = blockIdx.x * share;
    griddep_launch();
    if (w0 >= total) return;
    find_work(p, scan, per, before, mine, w0);
    if (warp == kStreams - 1) {
        if (lane == 0) {
            walk.left = min(total - w0, share);
            walk.b = scan.seq;
            walk.cached = -kSeqs;
            const int size = seq_of(p, scan.seq).recs + kItemCost;
            divide(scan.off, size, walk.item, walk.unit);
            if (p.whole && walk.unit) {                                 // the CTA has the items that start in its share
                walk.left -= size - walk.unit;
                walk.item++;
                walk.unit = 0;
            }
        }
        __syncwarp();
        next_item(p, walk, items[0]);
    }
    __syncthreads();
    uint8_t *my_ring = ring + stream * (ST * REC);
    uint32_t phase = 0;                                                 // of the stream's stages, one bit each
    // addresses of records k0 .. k0 + 31 of this stream, one per lane
    auto lookup = [&](const Item &it, int k0) -> unsigned long long {
        const int rec = it.ra + stream + (k0 + lane) * kStreams;
        return rec < it.rb ? (unsigned long long)kv4_record(p.c, it.b, (long long)rec * 16, it.h) : 0;
    };
    // 8 dimensions of a query row per thread and pass
    constexpr int QN = kRows * HD / 8 > kThreads ? kRows * HD / 8 / kThreads : 1;
    const int qc = tid % (HD / 8);
    auto load_q = [&](const Item &it, float (&x)[8], int pass) {
        const int qr = tid / (HD / 8) + pass * (kRows / QN);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = 0.0f;
        if (qr < it.valid) {
            const unsigned ri = it.tile * kRows + qr, tok = ri / group;
            load8(p.q, p.type, (it.row0 + (long long)tok) * p.q_stride + (long long)(it.h * group + (ri - tok * group)) * HD + qc * 8, x);
        }
    };

    unsigned long long addr = 0;
    bool lost = false;                        // a copy never came: this warp copies no more, its outputs are NaN
    float qx[QN][8];
    if (!items[0].none) {
        addr = lookup(items[0], 0);
#pragma unroll
        for (int i = 0; i < QN; i++) load_q(items[0], qx[i], i);
    }
    for (int cur = 0; !items[cur].none; cur ^= 1) {
        const Item &it = items[cur];
        const int ra = it.ra, all0 = it.all0, all1 = it.all1;
        const int nmine = lost ? 0 : max(0, (it.rb - ra - stream + kStreams - 1) / kStreams);    // records of this stream
        uint32_t there = 0;                 // stages that hold a record (not of a missing page)
        auto issue = [&](int k) {
            if (k >= nmine) return;
            if ((k & 31) == 0 && k) addr = lookup(it, k);
            const uint8_t *src = (const uint8_t *)__shfl_sync(0xffffffffu, addr, k & 31);
            const int st = k % ST;
            there = src ? there | 1u << st : there & ~(1u << st);
            if (src && lane == 0 && !(STARVE && blockIdx.x == 0 && stream == 0)) {
                mbar_arrive_expect_tx(&full[stream][st], REC);
                bulk_load(my_ring + st * REC, src, REC, &full[stream][st]);
            }
        };
        for (int k = 0; k < ST; k++) issue(k);
        if (warp == kStreams - 1) next_item(p, walk, items[cur ^ 1]);

        // query operands
#pragma unroll
        for (int pass = 0; pass < QN; pass++) {
            const float (&x)[8] = qx[pass];
            const int qr = tid / (HD / 8) + pass * (kRows / QN);
            float mx = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[i]));
#pragma unroll
            for (int o = 1; o < min(32, HD / 8); o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            if constexpr (HD / 8 > 32) {
                if (lane == 0) row_max[pass][warp] = mx;
                __syncthreads();
                mx = fmaxf(mx, row_max[pass][warp ^ 1]);
            }
            // exact power of two that brings the row's largest |q| to 2^13..2^14
            const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 115);
            // (the sign of the softmax scale goes with it, so that row_scale is positive)
            const float up = copysignf(__uint_as_float((uint32_t)(127 + 13 - e) << 23), p.scale);
            // 8 dimensions: group qc / 8, t = qc / 2 % 4, half qc % 2; steps 2 half + i take
            // dimensions 2i, 2i+4 and, a nibble up, 2i+1, 2i+5
            float rep = 0.0f;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float y[4] = {x[2 * i] * up, x[2 * i + 4] * up, x[2 * i + 1] * up * 0.0625f,
                                    x[2 * i + 5] * up * 0.0625f};
                hi[2 * i] = pack_h(y[0], y[1]);
                hi[2 * i + 1] = pack_h(y[2], y[3]);
                float2 f0 = unpack_h(hi[2 * i]), f1 = unpack_h(hi[2 * i + 1]);
                rep += f0.x + f0.y + 16.0f * (f1.x + f1.y);
                if (HILO) {
                    lo[2 * i] = pack_h(y[0] - f0.x, y[1] - f0.y);
                    lo[2 * i + 1] = pack_h(y[2] - f1.x, y[3] - f1.y);
                    f0 = unpack_h(lo[2 * i]);
                    f1 = unpack_h(lo[2 * i + 1]);
                    rep += f0.x + f0.y + 16.0f * (f1.x + f1.y);
                }
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) rep += __shfl_xor_sync(0xffffffffu, rep, o);
            if (qr < kRows) {
                if (qc == 0)
                    row_scale[qr] = fmaxf(fabsf(p.scale) * kLog2e * __uint_as_float((uint32_t)(127 + 24 - 13 + e) << 23),
                                          0x1p-120f);     // a scale of 0 still leaves -inf what it is
                const int to = ((qc >> 3) * 2 + (qc & 1)) * 32 + qr * 4 + (qc >> 1 & 3);
                qhi[to] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (HILO) qlo[to] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                if ((qc & 7) == 0) qoff[(qc >> 3) * 8 + qr] = -8.0f * 0x1p-24f * rep;
            }
        }
        __syncthreads();
        // this lane's row g sees the keys my_lo..my_hi
        const long long row_pos = it.pos0 + (it.tile * kRows + g) / group;
        const int cap = p.c.table_stride << p.c.page_shift;
        const int my_hi = g < it.valid ? (int)max(min(row_pos, (long long)cap - 1), -1ll) : -1;
        const int my_lo = p.window ? (int)min(max(row_pos - p.window + 1, 0ll), (long long)cap) : 0;

        float o[G][4][4];
#pragma unroll
        for (int i = 0; i < G; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[i][j][k] = 0.0f;
        float m = -INFINITY, l = 0.0f;
        const float rs = row_scale[g];

        uint32_t ph0 = 0, ph1 = 0, pl0 = 0, pl1 = 0;          // p of a record as high and low bf16
        uint64_t p01 = 0, p23 = 0;                            // with fp32 outputs: as it is
        uint32_t see01 = 0, see23 = 0;                        // which of its keys row g sees, as masks of the scales

        // scores of one group: lane holds keys g, g + 8 x rows 2t, 2t + 1
        auto score = [&](const uint8_t *rec, int gr, const uint32_t (&k0s)[(G + 1) / 2],
                         const uint32_t (&k1s)[(G + 1) / 2], float (&sc)[4]) {
            const uint4 kc = *reinterpret_cast<const uint4 *>(rec + gr * 512 + lane * 16);
            const float2 q0 = *reinterpret_cast<const float2 *>(qoff + gr * 8 + 2 * t);
            float d[4] = {q0.x, q0.y, q0.x, q0.y}, dl[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int half = 0; half < 2; half++) {
                uint32_t x = half ? kc.y : kc.x, z = half ? kc.w : kc.z;
                const int qi = (gr * 2 + half) * 32 + lane;
                const uint4 bh = qhi[qi];
                uint4 bl;
                if (HILO) bl = qlo[qi];
                const uint32_t a0 = x & 0x000f000fu, a1 = z & 0x000f000fu, a2 = x & 0x00f000f0u, a3 = z & 0x00f000f0u;
                mma_h(d, a0, a1, a2, a3, bh.x, bh.y);
                if (HILO) mma_h(dl, a0, a1, a2, a3, bl.x, bl.y);
                x >>= 8;
                z >>= 8;
                const uint32_t a4 = x & 0x000f000fu, a5 = z & 0x000f000fu, a6 = x & 0x00f000f0u, a7 = z & 0x00f000f0u;
                mma_h(d, a4, a5, a6, a7, bh.z, bh.w);
                if (HILO) mma_h(dl, a4, a5, a6, a7, bl.z, bl.w);
            }
            if (HILO) {
#pragma unroll
                for (int i = 0; i < 4; i++) d[i] += dl[i];
            }
            const float k0 = half_of(k0s[gr / 2], gr & 1), k1 = half_of(k1s[gr / 2], gr & 1);
            sc[0] = fmaf(d[0], k0, sc[0]);
            sc[1] = fmaf(d[1], k0, sc[1]);
            sc[2] = fmaf(d[2], k1, sc[2]);
            sc[3] = fmaf(d[3], k1, sc[3]);
        };
        // output of one group: lane holds dimensions 8g + 2j, + 1 x rows 2t, 2t + 1
        auto value = [&](const uint8_t *rec, int gr) {
            const uint4 vc = *reinterpret_cast<const uint4 *>(rec + 8 * HD + gr * 512 + lane * 16);
            uint2 vs = reinterpret_cast<const uint2 *>(rec + 16 * HD + 32 * G)[gr * 4 + t];
            vs.x &= see01;                                    // the scale of a token that is not seen may be anything
            vs.y &= see23;
            uint32_t h0, h1, l0, l1;                          // p vs = h + l
            if constexpr (HILO) {
                split(p01, vs.x, h0, l0);
                split(p23, vs.y, h1, l1);
            } else {
                // h the rounded product of p's high half, l what it lost and the low half's product
                h0 = mul_b(ph0, vs.x), h1 = mul_b(ph1, vs.y);
                l0 = fma_b(pl0, vs.x, fma_b(ph0, vs.x, h0 ^ 0x80008000u));
                l1 = fma_b(pl1, vs.y, fma_b(ph1, vs.y, h1 ^ 0x80008000u));
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t ab = __byte_perm(vc.x, vc.y, j < 2 ? 0x5410 : 0x7632) >> (8 * (j & 1));
                const uint32_t cd = __byte_perm(vc.z, vc.w, j < 2 ? 0x5410 : 0x7632) >> (8 * (j & 1));
                const uint32_t a0 = code_lo(ab), a1 = code_hi(ab), a2 = code_lo(cd), a3 = code_hi(cd);
                mma_b(o[gr][j], a0, a1, a2, a3, l0, l1);
                mma_b(o[gr][j], a0, a1, a2, a3, h0, h1);
            }
        };

        int st = 0;
        for (int k = 0; k < nmine; k++) {
            const uint8_t *rec = my_ring + st * REC;
            const bool here = there >> st & 1;                // a missing page has no keys
            if (here) {
                if (!__all_sync(0xffffffffu, mbar_wait(&full[stream][st], phase >> st & 1, nullptr, 0))) {
                    lost = true;                              // the others in flight are waited for, with the same limit
                    for (int i = 0; i < ST; i++)
                        if (there >> i & 1 && i != st) mbar_wait(&full[stream][i], phase >> i & 1, nullptr, 0);
                    break;
                }
                phase ^= 1u << st;
                float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                uint32_t k0s[(G + 1) / 2], k1s[(G + 1) / 2];  // scales of keys g and g + 8
                load_scales<G>(rec + 16 * HD + g * (2 * G), k0s);
                load_scales<G>(rec + 16 * HD + (g + 8) * (2 * G), k1s);
#pragma unroll
                for (int gr = 0; gr < G; gr++) score(rec, gr, k0s, k1s, sc);
                // row g, keys 2t, 2t + 1, 2t + 8, 2t + 9
                transpose2(sc[0], sc[1]);
                transpose2(sc[2], sc[3]);
                const int key0 = (ra + stream + k * kStreams) * 16;
                see01 = see23 = 0xffffffffu;
                if (key0 < all0 || key0 + 15 > all1) {
                    see01 = see23 = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int key = key0 + 2 * t + (i & 1) + 8 * (i >> 1);
                        const bool see = key >= my_lo && key <= my_hi;
                        if (!see) sc[i] = -INFINITY;
                        else if (i < 2) see01 |= 0xffffu << (16 * (i & 1));
                        else see23 |= 0xffffu << (16 * (i & 1));
                    }
                }
                float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * rs;
                // The reference m follows the maximum when that is kSlack above it: p stays
                // below 2^kSlack, and the outputs are rescaled a few times per sequence.
                if (__any_sync(0xffffffffu, mx > m + kSlack)) {
                    const float mn = mx > m + kSlack ? mx : m;
                    const float al = mn == -INFINITY ? 1.0f : ex2(m - mn);
                    m = mn;
                    l *= al;
                    const float al0 = __shfl_sync(0xffffffffu, al, 8 * t),
                                al1 = __shfl_sync(0xffffffffu, al, 8 * t + 4);
#pragma unroll
                    for (int i = 0; i < G; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            o[i][j][0] *= al0;
                            o[i][j][1] *= al1;
                            o[i][j][2] *= al0;
                            o[i][j][3] *= al1;
                        }
                }
                const float mref = m == -INFINITY ? 0.0f : m;
                float pr[4];
#pragma unroll
                for (int i = 0; i < 4; i++) pr[i] = ex2(fmaf(sc[i], rs, -mref));
                l += (pr[0] + pr[1]) + (pr[2] + pr[3]);
                // (not 80 more in the exponent, which would round it to 2^-18)
#pragma unroll
                for (int i = 0; i < 4; i++) pr[i] *= kUp;
                if constexpr (HILO) {
                    p01 = pk(pr[0], pr[1]);
                    p23 = pk(pr[2], pr[3]);
                } else {
                    ph0 = pack_b(pr[0], pr[1]);
                    ph1 = pack_b(pr[2], pr[3]);
                    pl0 = pack_b(pr[0] - half_of(ph0, 0), pr[1] - half_of(ph0, 1));
                    pl1 = pack_b(pr[2] - half_of(ph1, 0), pr[3] - half_of(ph1, 1));
                }
#pragma unroll
                for (int gr = 0; gr < G; gr++) value(rec, gr);
                __syncwarp();
            }
            issue(k + ST);                                    // into the stage that is free now
            st = st + 1 == ST ? 0 : st + 1;
        }
        if (lost) l = NAN;

        // ---- the warps meet; the next item's addresses and queries are on their way ----
        if (!items[cur ^ 1].none) {
            addr = lookup(items[cur ^ 1], 0);
#pragma unroll
            for (int i = 0; i < QN; i++) load_q(items[cur ^ 1], qx[i], i);
        }
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) { sm_m[stream][g] = m; sm_l[stream][g] = l; }
        __syncwarp();
        float *ow = reinterpret_cast<float *>(my_ring);
#pragma unroll
        for (int gr = 0; gr < G; gr++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int d = gr * 64 + 8 * g + 2 * j;
                *reinterpret_cast<float2 *>(ow + (2 * t) * C::kPad + d) =
                    make_float2(o[gr][j][0] * kEven, o[gr][j][2] * kOdd);
                *reinterpret_cast<float2 *>(ow + (2 * t + 1) * C::kPad + d) =
                    make_float2(o[gr][j][1] * kEven, o[gr][j][3] * kOdd);
            }
        __syncthreads();
        const int slot = 2 * blockIdx.x + (it.starts ? 1 : 0);
        // a thread finishes four pairs of a row, a warp 64 in a row at a time
        for (int r = tid / (HD / 8); r < kRows; r += kThreads / (HD / 8)) {
            float mt = sm_m[0][r];
#pragma unroll
            for (int k = 1; k < kStreams; k++) mt = fmaxf(mt, sm_m[k][r]);
            const float ref = mt == -INFINITY ? 0.0f : mt;
            float lt = 0.0f;
            float2 x[4] = {};
            const float *src = reinterpret_cast<const float *>(ring) + r * C::kPad + 2 * qc;
#pragma unroll
            for (int k = 0; k < kStreams; k++) {
                const float f = ex2(sm_m[k][r] - ref);
                lt = fmaf(f, sm_l[k][r], lt);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    constexpr int Q = HD / 4;
                    const float2 y = *reinterpret_cast<const float2 *>(
                        src + k * (ST * REC / 4) + j * Q);
                    x[j].x = fmaf(f, y.x, x[j].x);
                    x[j].y = fmaf(f, y.y, x[j].y);
                }
            }
            if (it.whole) {
                if (r < it.valid) {
                    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
                    const unsigned ri = it.tile * kRows + r, tok = ri / group;
                    const long long to = (it.row0 + (long long)tok) * p.out_stride +
                                         (long long)(it.h * group + (ri - tok * group)) * HD + 2 * qc;
#pragma unroll
                    for (int j = 0; j < 4; j++) store2(p.out, p.type, to + j * (HD / 4), x[j].x * inv, x[j].y * inv);
                }
            } else {
                if (qc == 0) {
                    p.stats[slot * (2 * kRows) + r] = mt;
                    p.stats[slot * (2 * kRows) + kRows + r] = lt;
                }
#pragma unroll
                for (int j = 0; j < 4; j++)
                    *reinterpret_cast<float2 *>(p.slots + (long long)slot * C::kSlot + r * HD + 2 * qc +
                                                j * (HD / 4)) = x[j];
            }
        }
        fence_async();                          // the ring is the copies' again
        __syncthreads();
    }
}

// Joins the partial results of the items that are cut between CTAs. Block c - 1
// looks at the cut at CTA c's start. The K - 1 blocks whose cuts lie in an item of
// K parts share its 8 x HD outputs evenly, so a block reads about one part's worth
// whether an item has two parts or 148.
template <int HD>
__global__ void __launch_bounds__(kJoinThreads) k_kv4_attn_join(const __grid_constant__ AttnP p) {
    using C = Cfg<HD>;
    constexpr int NV = kRows * HD / 8;                 // pieces of 8 outputs
    __shared__ Scan<kJoinThreads> scan;
    __shared__ float sm_f[C::kCtas * kRows], sm_l[C::kCtas * kRows], inv[kRows];
    const int c = blockIdx.x + 1, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (p.c.n + kJoinThreads - 1) / kJoinThreads;
    long long before, mine;
    const long long total = scan_total(p, scan, per, before, mine);
    const long long share = share_of(total, C::kCtas);
    const long long w = c * share;
    // Every block waits for the parts, also one with nothing to join: this grid's end is
    // what the next kernel of the stream goes by.
    if (w >= total) {
        griddep_wait();
        return;
    }
    find_work(p, scan, per, before, mine, w);
    const Seq s = seq_of(p, scan.seq);
    int item, inside;
    divide(scan.off, s.recs + kItemCost, item, inside);
    inside -= kItemCost;                               // records of the item before the cut
    if (inside <= 0) {                                 // not a cut
        griddep_wait();
        return;
    }
    const int tile = item / p.c.kv_heads, h = item % p.c.kv_heads;
    // CTAs c0, c0 + 1, ... hold the parts: the item's records are the units from w - inside on
    const int ahead = (int)min(share, 1ll << 30);
    const int c0 = c - (inside + ahead - 1) / ahead;
    const int parts = c - c0 + (s.recs - inside + ahead - 1) / ahead;
    const int nv = (NV + parts - 2) / (parts - 1);     // pieces of this block: [v0, v1)
    const int v0 = (c - c0 - 1) * nv, v1 = min(NV, v0 + nv);
    const unsigned group = p.group;
    auto slot = [&](int k) { return 2 * (c0 + k) + (k == 0); };
    griddep_wait();                                    // the schedule needs no partial result
    const int ra = v0 / (HD / 8), rn = max(0, (v1 - 1) / (HD / 8) - ra + 1);     // its rows
    for (int i = tid; i < parts * rn; i += kJoinThreads) {
        const int k = i / rn, r = ra + i % rn;
        sm_f[k * kRows + r] = p.stats[slot(k) * (2 * kRows) + r];
        sm_l[k * kRows + r] = p.stats[slot(k) * (2 * kRows) + kRows + r];
    }
    __syncthreads();
    if (warp < rn) {
        const int r = ra + warp;
        float mt = -INFINITY;
        for (int k = lane; k < parts; k += 32) mt = fmaxf(mt, sm_f[k * kRows + r]);
        mt = warp_max(mt);
        const float ref = mt == -INFINITY ? 0.0f : mt;
        float lt = 0.0f;
        for (int k = lane; k < parts; k += 32) {
            const float f = ex2(sm_f[k * kRows + r] - ref);
            sm_f[k * kRows + r] = f;
            lt = fmaf(f, sm_l[k * kRows + r], lt);
        }
        lt = warp_sum(lt);
        if (lane == 0) inv[r] = lt == 0.0f ? 0.0f : 1.0f / lt;
    }
    __syncthreads();
    // `width` lanes share a piece, up to five parts each loaded at once
    constexpr int kAtOnce = 5;
    int width = 1;
    while (width < 32 && width * kAtOnce < parts) width *= 2;
    const int sub = tid % width;
    for (int vb = v0; vb < v1; vb += kJoinThreads / width) {
        const int v = vb + tid / width, r = min(v, v1 - 1) / (HD / 8), d = min(v, v1 - 1) % (HD / 8) * 8;
        float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        for (int kb = 0; kb < parts; kb += kAtOnce * width) {
            float y[kAtOnce][8];
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const int k = kb + i * width + sub;
                if (k < parts) Kv4Vec<float>::load(p.slots + (long long)slot(k) * C::kSlot + r * HD + d, y[i]);
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const int k = kb + i * width + sub;
                const float f = k < parts ? sm_f[k * kRows + r] : 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (k < parts) x[j] = fmaf(f, y[i][j], x[j]);
            }
        }
        for (int o = 1; o < width; o <<= 1)
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] += __shfl_xor_sync(0xffffffffu, x[j], o);
        const unsigned ri = tile * kRows + r;
        if (sub == 0 && v < v1 && ri < (unsigned)s.q * group) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= inv[r];
            store8(p.out, p.type,
                   (s.row0 + (long long)(ri / group)) * p.out_stride + (long long)(h * group + ri % group) * HD + d, x);
        }
    }
}

template <int HD, bool HILO, bool STARVE = false>
cudaError_t launch_stream(const AttnP &p, cudaStream_t st) {
    using C = Cfg<HD>;
    constexpr auto kernel = k_kv4_attn<HD, HILO, STARVE>;
    const int smem = C::kRing + (HILO ? 2 : 1) * C::kQ + C::G * 32;
    cudaError_t e = g4_smem_optin((const void *)kernel, smem);
    if (e != cudaSuccess) return e;
    e = g4_launch(kernel, dim3(C::kCtas), dim3(kThreads), (size_t)smem, st, true, p);
    if (e != cudaSuccess || p.whole) return e;
    return g4_launch(k_kv4_attn_join<HD>, dim3(C::kCtas - 1), dim3(kJoinThreads), 0, st, true, p);
}

template <int HD>
cudaError_t launch_hd(AttnP &p, int starve, cudaStream_t st) {
    // Items of few records, not more of them than CTAs: a CTA has an item for itself, and the
    // second kernel is saved. One token of 8 heads and a window of 512 tokens (33 records), us
    // cut and whole: 64 dimensions, 1 / 64 / 128 sequences 9.7 / 7.7, 12.5 / 9.4, 16.4 / 9.8; 256
    // dimensions 13.6 / 13.0, 19.0 / 18.1, 23.2 / 19.2; 512 dimensions 17.5 / 18.1, 19.9 / 19.1,
    // 28.1 / 28.2. At 1000 tokens (63 records): 64 dimensions 9.7 / 9.7, 16.1 / 12.4, 18.4 / 12.7;
    // 256 dimensions 13.6 / 17.8, 23.1 / 26.3, 30.1 / 27.9.
    const long long cap = (long long)p.c.table_stride << p.c.page_shift,
                    seen = p.window && (long long)p.window + kRows < cap ? (long long)p.window + kRows : cap,
                    tiles = (long long)p.c.rows * p.group / kRows + p.c.n;
    p.whole = seen <= Cfg<HD>::kWhole * kKv4Rec && tiles * p.c.kv_heads <= Cfg<HD>::kCtas;
    p.stats = p.slots + (size_t)2 * Cfg<HD>::kCtas * Cfg<HD>::kSlot;
    if constexpr (HD >= 256)
        if (starve == 1 && p.type == G4_TYPE_F32) return launch_stream<HD, true, true>(p, st);
    if (starve) return cudaErrorNotSupported;
    return p.type == G4_TYPE_F32 ? launch_stream<HD, true>(p, st) : launch_stream<HD, false>(p, st);
}

template <int HD>
size_t ws_bytes() {
    return (size_t)2 * Cfg<HD>::kCtas * (Cfg<HD>::kSlot + 2 * kRows) * sizeof(float);
}

}  // namespace

size_t g4_kv4_attention_ws(const Kv4View &c, int type, int q_heads) {
    if (c.n == 0) return 16;
    // enough for every call of fewer rows, sequences or pages too, whichever kernel that takes
    const size_t few =
        c.hd == 64 ? ws_bytes<64>() : c.hd == 128 ? ws_bytes<128>() : c.hd == 256 ? ws_bytes<256>() : ws_bytes<512>();
    return std::max(few, kv4_prompt_ws(c, type, q_heads));
}

cudaError_t g4_launch_kv4_attention(const Kv4View &c, int type, int q_heads, const void *q, long long q_stride,
                                    void *out, long long out_stride, float scale, int window, void *ws, int starve,
                                    cudaStream_t st) {
    if (many_rows(c, q_heads))
        return kv4_launch_prompt(c, type, q_heads, q, q_stride, out, out_stride, scale, window, ws, starve, st);
    AttnP p;
    p.c = c;
    p.type = type;
    p.group = q_heads / c.kv_heads;
    p.q = q;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.scale = scale;
    p.window = window;
    p.slots = (float *)ws;
    if (c.hd == 64) return launch_hd<64>(p, starve, st);
    if (c.hd == 128) return launch_hd<128>(p, starve, st);
    if (c.hd == 256) return launch_hd<256>(p, starve, st);
    return launch_hd<512>(p, starve, st);
}
