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
//                -8 sum(q). q is scaled per row to 2^13..2^14 and, if fp32, split
//                into high and low halves (22 bits).
//   O^T = V^T P^T  bf16 (the scaled probabilities need its range): codes are
//                (128 + n) - 136, exact; p vs is split into high and low bf16
//                (16 bits).
// Every warp streams its own records of 16 keys through a ring in shared memory
// and keeps its own running maximum, sum and output; the warps meet once per
// sequence and head. Work is counted in records over all (sequence, row tile, kv
// head) and cut into one even run per CTA, so ragged batches and one long
// sequence fill the GPU alike; a sequence cut between CTAs leaves partial
// results that a second kernel joins in order.
#include <cuda_runtime.h>

#include "g4_kv4.cuh"

namespace {

constexpr int kRows = 8;          // query rows of a tile (tokens x heads of one kv head)
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kSms = 148;
constexpr float kLog2e = 1.4426950408889634f;

template <int HD>
struct Cfg {
    static constexpr int G = HD / kKv4Group;
    static constexpr int kRec = 17 * HD;
    static constexpr int kStages = HD == 512 ? 3 : HD == 256 ? 3 : HD == 128 ? 4 : 6;
    static constexpr int kOcc = HD == 512 ? 1 : 2;
    static constexpr int kCtas = kSms * kOcc;
    static constexpr int kRing = kWarps * kStages * kRec;
    static constexpr int kQ = G * 1024;                         // operands of the query tile (one half)
    static constexpr int kPad = HD + 8;                         // row of the warps' outputs when they meet
    static constexpr int kSlot = 2 * kRows + kRows * HD;        // floats of one partial result
    static_assert(kStages * kRec >= kRows * kPad * 4, "a warp's ring holds its output tile");
};

struct AttnP {
    Kv4View c;
    int type, group;              // query heads per kv head
    const void *q;
    void *out;
    long long q_stride, out_stride;
    float scale;
    int window;
    float *slots;                 // partial results, two per CTA
};

G4_DEV void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
G4_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
G4_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
// nibbles at bits [s, s + 4) of both halves -> the codes as bf16
G4_DEV uint32_t code_b(uint32_t x, int s) {
    const uint32_t w = ((x >> s) & 0x000f000fu) | 0x43004300u;      // 128 + n
    uint32_t y;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(w), "r"(0x43084308u));
    return y;
}
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

// ---- the schedule -------------------------------------------------------------
// Sequence b: its rows in tiles of kRows, each tile x kv head an item of `recs`
// records (those that the sequence's rows see between them; a tile skips what
// its own rows do not see; at least 1, so that empty rows are written).
struct Seq {
    int row0, q, tiles, recs, rec0;
    long long pos0;
};

G4_DEV Seq seq_of(const AttnP &p, int b) {
    Seq s;
    s.row0 = kv4_offset(p.c, b);
    s.q = max(kv4_offset(p.c, b + 1) - s.row0, 0);
    s.pos0 = p.c.start_pos[b];
    s.tiles = (int)(((long long)s.q * p.group + kRows - 1) / kRows);
    const long long lo = p.window ? max(s.pos0 - p.window + 1, 0ll) : 0;
    const long long hi = min(s.pos0 + s.q - 1, ((long long)p.c.table_stride << p.c.page_shift) - 1);
    s.rec0 = (int)(lo >> 4);
    s.recs = hi < lo ? 1 : (int)((hi >> 4) - (lo >> 4)) + 1;
    return s;
}
G4_DEV long long work_of(const AttnP &p, const Seq &s) { return (long long)s.tiles * p.c.kv_heads * s.recs; }

// Total work, and where unit `w` of it lies: sequence and offset in its work.
// Every thread of a block of N calls it; `s` is shared memory.
struct Where {
    long long total, off;
    int seq;
};
template <int N>
struct Scan {
    long long warp[N / 32], off;
    int seq;
};
template <int N>
G4_DEV long long scan_total(const AttnP &p, Scan<N> &s, int per, long long &before, long long &mine) {
    const int tid = threadIdx.x, lane = tid & 31;
    mine = 0;
    for (int b = tid * per; b < min((tid + 1) * per, p.c.n); b++) mine += work_of(p, seq_of(p, b));
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) s.warp[tid >> 5] = inc;
    __syncthreads();
    long long total = 0, base = 0;
    for (int i = 0; i < N / 32; i++) {
        if (i < (tid >> 5)) base += s.warp[i];
        total += s.warp[i];
    }
    before = base + inc - mine;
    return total;
}
template <int N>
G4_DEV Where find_work(const AttnP &p, Scan<N> &s, int per, long long total, long long before, long long mine,
                       long long w) {
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
    return {total, s.off, s.seq};
}
G4_DEV long long share_of(long long total, int ctas) { return max((total + ctas - 1) / ctas, (long long)kWarps); }

// ---- the streaming kernel -------------------------------------------------------
template <int HD, bool HILO>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::kOcc) k_kv4_attn(const __grid_constant__ AttnP p) {
    using C = Cfg<HD>;
    constexpr int G = C::G, REC = C::kRec, ST = C::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;
    uint4 *qhi = reinterpret_cast<uint4 *>(smem + C::kRing);            // [G][2][32] (lane's operands of two steps)
    uint4 *qlo = qhi + C::kQ / 16;
    float *qoff = reinterpret_cast<float *>(smem + C::kRing + (HILO ? 2 : 1) * C::kQ);   // [G][8]: -8 sum q
    __shared__ Scan<kThreads> scan;
    __shared__ float row_scale[kRows], sm_m[kWarps][kRows], sm_l[kWarps][kRows];
    __shared__ int sm_ok[kWarps][8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int group = p.group, kvh = p.c.kv_heads;
    const long long cap = (long long)p.c.table_stride << p.c.page_shift;

    const int per = (p.c.n + kThreads - 1) / kThreads;
    long long before, mine;
    const long long total = scan_total(p, scan, per, before, mine);
    const long long share = share_of(total, C::kCtas);
    const long long w0 = blockIdx.x * share, w1 = min(total, w0 + share);
    if (w0 >= w1) return;
    const Where at = find_work(p, scan, per, total, before, mine, w0);
    int b = at.seq;
    long long off = at.off;
    uint8_t *my_ring = ring + warp * (ST * REC);

    for (long long w = w0; w < w1;) {
        const Seq s = seq_of(p, b);
        const long long work = work_of(p, s);
        if (off >= work) {          // next sequence (empty ones have no work)
            off -= work;
            b++;
            continue;
        }
        const int item = (int)(off / s.recs), r0 = (int)(off % s.recs);
        const int r1 = (int)min((long long)s.recs, r0 + (w1 - w));
        const int tile = item / kvh, h = item % kvh;
        const bool whole = r0 == 0 && r1 == s.recs;
        const bool starts = r0 == 0;
        w += r1 - r0;
        off += r1 - r0;

        // what the tile's rows see: rows are (token, head of the group), token-major
        const long long rows_left = (long long)s.q * group - (long long)tile * kRows;
        const int valid = (int)min(rows_left, (long long)kRows);
        const long long tok0 = (long long)tile * kRows / group, tok1 = ((long long)tile * kRows + valid - 1) / group;
        const long long pos_first = s.pos0 + tok0, pos_last = s.pos0 + tok1;
        const long long see0 = p.window ? max(pos_first - p.window + 1, 0ll) : 0;       // any row sees [see0, see1]
        const long long see1 = min(pos_last, cap - 1);
        const long long all0 = p.window ? max(pos_last - p.window + 1, 0ll) : 0;        // every row sees [all0, pos_first]
        const int ra = max(s.rec0 + r0, (int)(see0 >> 4));
        const int rb = see1 < see0 ? ra : min(s.rec0 + r1, (int)(see1 >> 4) + 1);
        const int nmine = max(0, (rb - ra - warp + kWarps - 1) / kWarps);               // records of this warp
        // this lane's row g
        const long long idx = (long long)tile * kRows + g;
        const long long row_pos = s.pos0 + idx / group;
        const int my_hi = g < valid ? (int)max(min(row_pos, cap - 1), -1ll) : -1;
        const int my_lo = p.window ? (int)min(max(row_pos - p.window + 1, 0ll), cap) : 0;

        // addresses of the next 32 of this warp's records, one per lane
        unsigned long long addr = 0;
        auto lookup = [&](int k0) {
            const int k = k0 + lane;
            addr = 0;
            if (k < nmine)
                addr = (unsigned long long)kv4_record(p.c, b, (long long)(ra + warp + k * kWarps) * 16, h);
        };
        auto issue = [&](int k) {
            if (k < nmine) {
                if ((k & 31) == 0) lookup(k);
                const uint8_t *src = (const uint8_t *)__shfl_sync(0xffffffffu, addr, k & 31);
                if (lane == 0) sm_ok[warp][k % ST] = src != nullptr;
                if (src) {
                    const uint32_t dst = smem_u32(my_ring + (k % ST) * REC);
#pragma unroll
                    for (int i = 0; i < (REC / 16 + 31) / 32; i++)
                        if (i * 32 + lane < REC / 16) cp16(dst + (i * 32 + lane) * 16, src + (i * 32 + lane) * 16);
                }
            }
            cp_commit();
        };
        for (int k = 0; k < ST - 1; k++) issue(k);

        // query operands: warp r prepares row r, 8 dimensions a lane
        __syncthreads();            // the previous item's operands are no longer read
        {
            const int r = warp;
            const long long ri = (long long)tile * kRows + r;
            const long long at_q = (s.row0 + ri / group) * p.q_stride + (long long)(h * group + ri % group) * HD;
            constexpr int NC = (HD / 8 + 31) / 32;
            float x[NC][8], mx = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[c][i] = 0.0f;
                if (r < valid && c * 32 + lane < HD / 8) load8(p.q, p.type, at_q + (c * 32 + lane) * 8, x[c]);
#pragma unroll
                for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[c][i]));
            }
            mx = warp_max(mx);
            // exact power of two that brings the row's largest |q| to 2^13..2^14
            const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 115);
            const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
            if (lane == 0) row_scale[r] = p.scale * kLog2e * __uint_as_float((uint32_t)(127 + 24 - 13 + e) << 23);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int ch = c * 32 + lane;             // chunk of 8 dimensions: group ch / 8, t = ch / 2 % 4, half ch % 2
                float rep = 0.0f;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 2; i++) {             // steps 2 half + i: dimensions 2i, 2i+4 and (a nibble up) 2i+1, 2i+5
                    const float y[4] = {x[c][2 * i] * up, x[c][2 * i + 4] * up, x[c][2 * i + 1] * up * 0.0625f,
                                        x[c][2 * i + 5] * up * 0.0625f};
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
                if (ch < HD / 8) {
                    const int to = ((ch >> 3) * 2 + (ch & 1)) * 32 + r * 4 + (ch >> 1 & 3);
                    qhi[to] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (HILO) qlo[to] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    if ((ch & 7) == 0) qoff[(ch >> 3) * 8 + r] = -8.0f * 0x1p-24f * rep;
                }
            }
        }
        __syncthreads();

        float o[G][4][4];
#pragma unroll
        for (int i = 0; i < G; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[i][j][k] = 0.0f;
        float m = -INFINITY, l = 0.0f;
        const float rs0 = row_scale[2 * t], rs1 = row_scale[2 * t + 1];

        for (int k = 0; k < nmine; k++) {
            cp_wait<ST - 2>();
            __syncwarp();
            issue(k + ST - 1);
            if (!sm_ok[warp][k % ST]) continue;           // no page: no keys
            const uint8_t *rec = my_ring + (k % ST) * REC;
            const int key0 = (ra + warp + k * kWarps) * 16;

            // ---- scores: lane holds keys g, g + 8 x rows 2t, 2t + 1 ----
            float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const uint16_t *ks = reinterpret_cast<const uint16_t *>(rec + 16 * HD) + g * G;
#pragma unroll
            for (int gr = 0; gr < G; gr++) {
                const uint4 kc = *reinterpret_cast<const uint4 *>(rec + gr * 512 + lane * 16);
                const float2 q0 = *reinterpret_cast<const float2 *>(qoff + gr * 8 + 2 * t);
                float d[4] = {q0.x, q0.y, q0.x, q0.y};
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    uint32_t x = half ? kc.y : kc.x, z = half ? kc.w : kc.z;
                    const uint4 bh = qhi[(gr * 2 + half) * 32 + lane];
                    uint4 bl;
                    if (HILO) bl = qlo[(gr * 2 + half) * 32 + lane];
                    const uint32_t a0 = x & 0x000f000fu, a1 = z & 0x000f000fu, a2 = x & 0x00f000f0u,
                                   a3 = z & 0x00f000f0u;
                    mma_h(d, a0, a1, a2, a3, bh.x, bh.y);
                    if (HILO) mma_h(d, a0, a1, a2, a3, bl.x, bl.y);
                    x >>= 8;
                    z >>= 8;
                    const uint32_t a4 = x & 0x000f000fu, a5 = z & 0x000f000fu, a6 = x & 0x00f000f0u,
                                   a7 = z & 0x00f000f0u;
                    mma_h(d, a4, a5, a6, a7, bh.z, bh.w);
                    if (HILO) mma_h(d, a4, a5, a6, a7, bl.z, bl.w);
                }
                const float k0 = bf16_bits_f(ks[gr]), k1 = bf16_bits_f(ks[8 * G + gr]);
                sc[0] = fmaf(d[0], k0, sc[0]);
                sc[1] = fmaf(d[1], k0, sc[1]);
                sc[2] = fmaf(d[2], k1, sc[2]);
                sc[3] = fmaf(d[3], k1, sc[3]);
            }
            sc[0] *= rs0;
            sc[1] *= rs1;
            sc[2] *= rs0;
            sc[3] *= rs1;
            // ---- row g, keys 2t, 2t + 1, 2t + 8, 2t + 9 ----
            transpose2(sc[0], sc[1]);
            transpose2(sc[2], sc[3]);
            const bool edge = key0 < all0 || key0 + 15 > pos_first;
            bool see[4];
            if (edge) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int key = key0 + 2 * t + (i & 1) + 8 * (i >> 1);
                    see[i] = key >= my_lo && key <= my_hi;
                    if (!see[i]) sc[i] = -INFINITY;
                }
            }
            float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (__any_sync(0xffffffffu, mx > m)) {
                const float mn = fmaxf(m, mx);
                const float al = mn == -INFINITY ? 1.0f : ex2(m - mn);
                m = mn;
                l *= al;
                const float al0 = __shfl_sync(0xffffffffu, al, 8 * t), al1 = __shfl_sync(0xffffffffu, al, 8 * t + 4);
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
            for (int i = 0; i < 4; i++) pr[i] = ex2(sc[i] - mref);
            l += (pr[0] + pr[1]) + (pr[2] + pr[3]);

            // ---- output: lane holds dimensions 8g + 2j, + 1 of each group x rows 2t, 2t + 1 ----
            const uint2 *vsp = reinterpret_cast<const uint2 *>(rec + 16 * HD + 32 * G) + t;
#pragma unroll
            for (int gr = 0; gr < G; gr++) {
                const uint4 vc = *reinterpret_cast<const uint4 *>(rec + 8 * HD + gr * 512 + lane * 16);
                const uint2 vs = vsp[gr * 4];
                float pv[4] = {pr[0] * __uint_as_float(vs.x << 16), pr[1] * __uint_as_float(vs.x & 0xffff0000u),
                               pr[2] * __uint_as_float(vs.y << 16), pr[3] * __uint_as_float(vs.y & 0xffff0000u)};
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!see[i]) pv[i] = 0.0f;        // the scale of a token that is not there may be anything
                }
                const uint32_t h0 = pack_b(pv[0], pv[1]), h1 = pack_b(pv[2], pv[3]);
                const uint32_t l0 = pack_b(pv[0] - __uint_as_float(h0 << 16), pv[1] - __uint_as_float(h0 & 0xffff0000u));
                const uint32_t l1 = pack_b(pv[2] - __uint_as_float(h1 << 16), pv[3] - __uint_as_float(h1 & 0xffff0000u));
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const uint32_t ab = __byte_perm(vc.x, vc.y, half ? 0x7632 : 0x5410);
                    const uint32_t cd = __byte_perm(vc.z, vc.w, half ? 0x7632 : 0x5410);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint32_t a0 = code_b(ab, 8 * i), a1 = code_b(ab, 8 * i + 4), a2 = code_b(cd, 8 * i),
                                       a3 = code_b(cd, 8 * i + 4);
                        mma_b(o[gr][2 * half + i], a0, a1, a2, a3, h0, h1);
                        mma_b(o[gr][2 * half + i], a0, a1, a2, a3, l0, l1);
                    }
                }
            }
        }
        cp_wait<0>();
        __syncwarp();

        // ---- the warps meet ----
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) { sm_m[warp][g] = m; sm_l[warp][g] = l; }
        float *ow = reinterpret_cast<float *>(my_ring);
#pragma unroll
        for (int gr = 0; gr < G; gr++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int d = gr * 64 + 8 * g + 2 * j;
                *reinterpret_cast<float2 *>(ow + (2 * t) * C::kPad + d) = make_float2(o[gr][j][0], o[gr][j][2]);
                *reinterpret_cast<float2 *>(ow + (2 * t + 1) * C::kPad + d) = make_float2(o[gr][j][1], o[gr][j][3]);
            }
        __syncthreads();
        float *slot = p.slots + (long long)(2 * blockIdx.x + (starts ? 1 : 0)) * C::kSlot;
        for (int i = tid; i < kRows * HD / 8; i += kThreads) {
            const int r = i / (HD / 8), d = i % (HD / 8) * 8;
            float mt = sm_m[0][r];
#pragma unroll
            for (int k = 1; k < kWarps; k++) mt = fmaxf(mt, sm_m[k][r]);
            const float ref = mt == -INFINITY ? 0.0f : mt;
            float lt = 0.0f, x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < kWarps; k++) {
                const float f = ex2(sm_m[k][r] - ref);
                lt = fmaf(f, sm_l[k][r], lt);
                const float *src = reinterpret_cast<const float *>(ring + k * (ST * REC)) + r * C::kPad + d;
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = fmaf(f, src[j], x[j]);
            }
            if (whole) {
                if (r < valid) {
                    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] *= inv;
                    const long long ri = (long long)tile * kRows + r;
                    store8(p.out, p.type,
                           (s.row0 + ri / group) * p.out_stride + (long long)(h * group + ri % group) * HD + d, x);
                }
            } else {
                if (d == 0) {
                    slot[r] = mt;
                    slot[kRows + r] = lt;
                }
                Kv4Vec<float>::store(slot + 2 * kRows + r * HD + d, x);
            }
        }
        __syncthreads();
    }
}

// Joins the partial results of an item that CTAs c - 1, c, ... share. Block
// (c, r) does row r of the item that is cut at CTA c's start, if c is the first
// CTA to start inside it.
template <int HD>
__global__ void __launch_bounds__(128) k_kv4_attn_join(const __grid_constant__ AttnP p) {
    using C = Cfg<HD>;
    __shared__ Scan<128> scan;
    griddep_wait();
    const int c = blockIdx.x + 1, r = blockIdx.y, tid = threadIdx.x;
    const int per = (p.c.n + 127) / 128;
    long long before, mine;
    const long long total = scan_total(p, scan, per, before, mine);
    const long long share = share_of(total, C::kCtas);
    const long long w = c * share;
    if (w >= total) return;
    const Where at = find_work(p, scan, per, total, before, mine, w);
    const Seq s = seq_of(p, at.seq);
    const int item = (int)(at.off / s.recs), inside = (int)(at.off % s.recs);
    if (inside == 0 || inside > share) return;        // not cut here, or cut before too
    const int tile = item / p.c.kv_heads, h = item % p.c.kv_heads;
    const long long ri = (long long)tile * kRows + r;
    if (ri >= (long long)s.q * p.group) return;
    const long long end = w - inside + s.recs;        // first unit behind the item
    const int last = (int)((end - 1) / share);        // CTAs c - 1 .. last hold parts
    const float *first = p.slots + (long long)(2 * (c - 1) + 1) * C::kSlot;
    auto part = [&](int k) { return k == c - 1 ? first : p.slots + (long long)(2 * k) * C::kSlot; };
    float mt = -INFINITY;
    for (int k = c - 1; k <= last; k++) mt = fmaxf(mt, part(k)[r]);
    const float ref = mt == -INFINITY ? 0.0f : mt;
    const long long at_out = (s.row0 + ri / p.group) * p.out_stride + (long long)(h * p.group + ri % p.group) * HD;
    for (int d = tid * 8; d < HD; d += 128 * 8) {
        float lt = 0.0f, x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int k = c - 1; k <= last; k++) {
            const float *q = part(k);
            const float f = ex2(q[r] - ref);
            float y[8];
            Kv4Vec<float>::load(q + 2 * kRows + r * HD + d, y);
            lt = fmaf(f, q[kRows + r], lt);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = fmaf(f, y[j], x[j]);
        }
        const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] *= inv;
        store8(p.out, p.type, at_out + d, x);
    }
}

template <int HD, bool HILO>
cudaError_t launch_stream(const AttnP &p, cudaStream_t st) {
    using C = Cfg<HD>;
    const int smem = C::kRing + (HILO ? 2 : 1) * C::kQ + C::G * 32;
    cudaError_t e = g4_smem_optin((const void *)k_kv4_attn<HD, HILO>, smem);
    if (e != cudaSuccess) return e;
    e = g4_launch(k_kv4_attn<HD, HILO>, dim3(C::kCtas), dim3(kThreads), (size_t)smem, st, false, p);
    if (e != cudaSuccess) return e;
    return g4_launch(k_kv4_attn_join<HD>, dim3(C::kCtas - 1, kRows), dim3(128), 0, st, true, p);
}

template <int HD>
cudaError_t launch_hd(const AttnP &p, cudaStream_t st) {
    return p.type == G4_TYPE_F32 ? launch_stream<HD, true>(p, st) : launch_stream<HD, false>(p, st);
}

template <int HD>
size_t ws_bytes() {
    return (size_t)2 * Cfg<HD>::kCtas * Cfg<HD>::kSlot * sizeof(float);
}

}  // namespace

size_t g4_kv4_attention_ws(const Kv4View &c, int, int) {
    return c.hd == 64 ? ws_bytes<64>() : c.hd == 128 ? ws_bytes<128>() : c.hd == 256 ? ws_bytes<256>() : ws_bytes<512>();
}

cudaError_t g4_launch_kv4_attention(const Kv4View &c, int type, int q_heads, const void *q, long long q_stride,
                                    void *out, long long out_stride, float scale, int window, void *ws,
                                    cudaStream_t st) {
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
    if (c.hd == 64) return launch_hd<64>(p, st);
    if (c.hd == 128) return launch_hd<128>(p, st);
    if (c.hd == 256) return launch_hd<256>(p, st);
    return launch_hd<512>(p, st);
}
