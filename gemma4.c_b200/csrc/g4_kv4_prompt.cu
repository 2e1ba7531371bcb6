// g4_kv4_prompt.cu — attention over the paged 4-bit KV cache for many query rows
// of a sequence (prompts, chunks): tcgen05 GEMMs on tiles of 128 rows x 64 keys.
//
// With many rows per key the two products dominate (4 x rows x keys x hd FLOP), so
// they run on the 5th-generation tensor cores, and what would otherwise cost as
// much, turning 4-bit codes into operands, is done once per 128 rows:
//   S = Q K^T   fp16 operands in shared memory, fp32 accumulator in TMEM
//   O += P V    P (fp16) in TMEM as the A operand, V^T in shared memory
// Operands: a key or value c * scale has 11 significant bits (8 of the scale, 3 of
// the code), so as fp16 it is exact once the largest scale of the keys in work (of values:
// in their group of dimensions) is brought to a fixed power of two (of scales below 2^-11 of
// the largest, bits are lost that are 2^-20 of the largest value at most). q is scaled per row by a power of two; an fp32 q
// is split into high and low fp16 (22 bits; one fp16 holds a 16-bit q exactly), and so is
// p for every type (one fp16 p, 11 bits, would show beside an fp16 output's own rounding).
//
// A CTA has one accumulator of 128 rows x 256 dimensions, all that TMEM holds beside
// two S and two P tiles. 512 dimensions take a cluster of two CTAs, each with half
// of the dimensions of q, K and V: they exchange their halves of S through
// distributed shared memory, so that neither product is done twice.
// Roles of the 17 warps: 0-7 softmax (two threads per row = TMEM lane, 32 keys each),
// 8-15 conversion (each a record of the tile and some of its groups, the next tile's
// codes in flight in registers), 16 the MMAs. S and P are double-buffered: while the softmax works on tile
// j, the MMAs of P_{j-1} V and S_{j+1} run and K of tile j + 2 and V of tile j are converted.
//
// Measured: 512 tokens of 8 fp32 heads of 512 dimensions behind 15872 451 us (300 TFLOP/s
// of the operator's, twice that on the tensor cores, which work on two terms of q and of
// p); 2048 tokens of 256 dimensions behind 6144 297 us (405); 2048 tokens of 32 bf16 heads
// of 128 dimensions, 8 kv heads, 110 us (312). A tile takes 3.2 us at 512 dimensions, where
// the MMAs need 1.4 and sending the halves of S (32 KB each way, st.async; plain remote
// stores with one arrival a warp 522 us, sending before the maximum 463 us) bounds it; 2.1 us
// at 256, where MMAs of 64 columns (48 clocks against 32 for their share) bound it.
#include <algorithm>
#include <atomic>

#include <cuda_runtime.h>

#include "g4_kv4.cuh"
#include "g4_tc.cuh"

namespace {

constexpr int kM = 128;            // query rows of a tile
constexpr int kT = 64;             // keys of a tile: 4 records
constexpr int kH = kT / 2;         // keys of a softmax thread
constexpr int kSoftWarps = 8, kConvWarps = 8;
constexpr int kThreads = (kSoftWarps + kConvWarps + 1) * 32;
// Registers: five warps on one of an SM's four parts leave 96 a thread, on which the
// softmax spilled in its loop (chunk of 512 tokens at 16384: 532 us). The conversion
// gives it some of its own: 455 us.
constexpr int kRegs = 96, kSoftRegs = 112, kConvRegs = 80;
static_assert(kSoftWarps * kSoftRegs + kConvWarps * kConvRegs <= (kSoftWarps + kConvWarps) * kRegs,
              "the block has what its warps take");
constexpr int kSms = 148;
constexpr int kJoinThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
// The reference m of a row starts kHead above its first maximum and moves when the
// maximum is kSlack above it, that is after growing by 2^7.9; p is 2^14 times too large.
// So its halves stay below 65504, and p has steps of 2^-32 of the largest at most
// (with a growth of 2^4 between rescalings two tiles in three had one, 0.8 us each).
constexpr float kHead = 6.0f, kSlack = 1.9f, kUp = 14.0f;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256;      // TMEM columns: 2 x 64, 2 x (32 + 32), 256

template <int HD, bool HILO>
struct Cfg {
    static constexpr int kDc = HD > 256 ? 256 : HD;          // dimensions of a CTA
    static constexpr int kCl = HD / kDc;                     // CTAs of a cluster
    static constexpr int G = kDc / kKv4Group;
    static constexpr int kQ = G * kM * 128;                  // one half of q: G tiles of 128 rows x 128 bytes
    static constexpr int kK = G * kT * 128;
    static constexpr int kV = kDc * 128;                     // V^T: rows are dimensions, 64 keys
    // The tensor cores truncate as they add up, 8 steps a tile: an error that grows with
    // the length of a run (fp32, 128 tiles: 2e-5 of the output, 5e-5 where values have one
    // sign; after 32 tiles 5.3e-6 and 1.1e-5, after 16 3.3e-6 and 5.6e-6). So O is added to a
    // sum in memory, in fp32, after every kRun tiles (chunk of 512 tokens at 16384 without
    // sums 414 us, every 32 tiles 438, every 16 451).
    // 16-bit outputs round by more than that up to 256.
    static constexpr int kRun = HILO ? 16 : 256;
    static constexpr int kX = kCl > 1 ? kM * kT * 4 : 0;     // the other CTA's half of S
    static constexpr int kSmem = kQ * (HILO ? 2 : 1) + kK + kV + kX;
};

struct PromptP {
    Kv4View c;
    int type;
    unsigned group;                // query heads per kv head
    int tokens;                    // per tile: 128 / group
    int slots, splits;             // row tiles (an upper bound), key ranges of each
    const void *q;
    void *out;
    long long q_stride, out_stride;
    float scale;
    int window;
    int starve;                    // of a STARVE kernel: 1 K of block 0 is never announced, 2 a wait there counts as run out
    float *parts, *stats;          // [slots][kv heads][splits][HD / 4][128][4], [..][2][128]
};

G4_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
G4_DEV uint32_t pack_h(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
G4_DEV float2 unpack_h(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
G4_DEV uint32_t fma_h(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t y;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(a), "r"(b), "r"(c));
    return y;
}
G4_DEV uint32_t mul_h(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
// 2^e as fp32, e in -126..127
G4_DEV float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
G4_DEV void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
G4_DEV uint32_t rank_addr(uint32_t addr, uint32_t rank) {
    uint32_t y;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(y) : "r"(addr), "r"(rank));
    return y;
}
// 16 bytes into the other CTA's shared memory, counted on its barrier
G4_DEV void remote_store4(uint32_t addr, float x, float y, float z, float w, uint32_t bar) {
    asm volatile(
        "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr),
        "f"(x), "f"(y), "f"(z), "f"(w), "r"(bar)
        : "memory");
}
G4_DEV void remote_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
G4_DEV void remote_store(uint32_t addr, int x) {
    asm volatile("st.relaxed.cluster.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(x) : "memory");
}
G4_DEV bool wait_cluster(uint64_t *bar, uint32_t parity) {       // bounded, like mbar_wait
    const uint64_t t0 = g4_globaltimer();
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
            " selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if (g4_globaltimer() - t0 > G4_WAIT_NS) return false;
    }
}
G4_DEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
G4_DEV void mma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(db), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
G4_DEV void tmem_st32(uint32_t taddr, const int (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
G4_DEV void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
G4_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Four values added to memory without waiting for them
G4_DEV void red_add4(float *p, float x, float y, float z, float w) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(x), "f"(y), "f"(z), "f"(w)
                 : "memory");
}

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

// ---- what a tile of rows sees ---------------------------------------------------
// Row tiles: sequence b has the slots [offsets[b] / tokens + b, offsets[b + 1] / tokens
// + b + 1), at least as many as its tiles of `tokens` tokens.
struct Item {
    int seq, row0, tok0, tokens;       // sequence, its first row, first token and tokens of the tile
    long long pos0;                    // position of the sequence's first row
    int see0, see1;                    // keys that some row sees (see1 < see0: none)
    int all0, all1;                    // keys that every row sees
};
G4_DEV int slot_base(const PromptP &p, int b) { return kv4_offset(p.c, b) / p.tokens + b; }
G4_DEV bool find_item(const PromptP &p, int slot, Item &it) {
    int lo = 0, hi = p.c.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (slot_base(p, mid) <= slot) lo = mid;
        else hi = mid;
    }
    it.seq = lo;
    it.row0 = kv4_offset(p.c, lo);
    const int q = kv4_offset(p.c, lo + 1) - it.row0;
    const int i = slot - slot_base(p, lo);
    if (i < 0 || q <= 0 || i >= (q + p.tokens - 1) / p.tokens) return false;
    it.tok0 = i * p.tokens;
    it.tokens = min(p.tokens, q - it.tok0);
    it.pos0 = p.c.start_pos[lo];
    const long long cap = (long long)p.c.table_stride << p.c.page_shift, first = it.pos0 + it.tok0,
                    last = first + it.tokens - 1;
    it.see0 = p.window ? (int)min(max(first - p.window + 1, 0ll), cap) : 0;
    it.see1 = (int)max(min(last, cap - 1), -1ll);
    it.all0 = p.window ? (int)min(max(last - p.window + 1, 0ll), cap) : 0;
    it.all1 = (int)max(min(first, cap - 1), -1ll);
    return true;
}
// Key tiles of split s: [t0, t1)
G4_DEV void tiles_of(const Item &it, int s, int splits, int &t0, int &t1) {
    if (it.see1 < it.see0) {
        t0 = t1 = 0;
        return;
    }
    const int a = it.see0 / kT, n = it.see1 / kT + 1 - a;
    t0 = a + (int)((long long)n * s / splits);
    t1 = a + (int)((long long)n * (s + 1) / splits);
}

// Two codes (nibbles of the halves' bits m) times their scales: n 2^-21 or n 2^-17 (a
// subnormal) times S, less 8 S: exact.
G4_DEV uint32_t value2(uint32_t x, uint32_t mask, uint32_t s, uint32_t off) { return fma_h(x & mask, s, off); }
// A scale for that: keys that no row of the tile sees may have larger ones than were
// looked for, or whatever an unwritten slot holds; they only have to stay finite (an
// operand of 0 times infinity is NaN). NaN stays NaN.
G4_DEV float bound(float f) { return f > 4080.0f ? 4080.0f : f < -4080.0f ? -4080.0f : f; }
constexpr uint32_t kLoMask = 0x00780078u, kHiMask = 0x07800780u;

// STARVE: the test aid g4_test_kv4_attention_starve.
template <int HD, bool HILO, bool STARVE>
__global__ void __launch_bounds__(kThreads, 1) k_kv4_prompt(const __grid_constant__ PromptP p) {
    using C = Cfg<HD, HILO>;
    constexpr int G = C::G, HG = HD / kKv4Group, DC = C::kDc, CL = C::kCl;
    constexpr int NB = G > 1 ? G / 2 : 1;                       // groups of a conversion warp
    extern __shared__ __align__(1024) uint8_t base[];          // tiles with the 128-byte swizzle
    __shared__ uint64_t kfull, vfull, ended, sfull[2], pfull[2], odone[2];
    __shared__ uint64_t xfull[kSoftWarps], xfree[kSoftWarps];   // a softmax warp and its like in the other CTA
    __shared__ uint32_t tmem_slot;
    __shared__ float pair[2][2][kM];                            // between the two threads of a row
    // 1 / power of two of each row's q: read by both threads of a row before they first meet,
    // and so before tile 1 writes here
    float *q_inv = pair[1][0];
    __shared__ uint32_t k_top, v_top[G];                        // largest scales (bf16 bits) of the keys in work
    __shared__ int missing[4][4];                               // [tile % 4][record]: tile + 1 if its page is missing
    __shared__ int nan_tile[4];                                 // [tile % 4]: tile + 1 if a value of it is NaN
    __shared__ int2 nan_keys[4][G][4];                          // [tile % 4][group][record]: tile + 1, keys
    __shared__ int failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CL > 1 ? blockIdx.x % CL : 0;
    uint8_t *qh = base, *ql = qh + (HILO ? C::kQ : 0), *kb = ql + C::kQ, *vb = kb + C::kK;
    float4 *xb = reinterpret_cast<float4 *>(vb + C::kV);        // [16][128]: 4 keys x rows

    griddep_wait();
    const int id = blockIdx.x / CL;
    const int split = id % p.splits, hs = id / p.splits, h = hs % p.c.kv_heads;
    const int slot = p.slots - 1 - hs / p.c.kv_heads;           // the longest rows of a prompt first
    Item it;
    if (!find_item(p, slot, it)) return;                        // the same for the whole cluster
    int t0, t1;
    tiles_of(it, split, p.splits, t0, t1);
    const int nt = t1 - t0;
    // O is summed up in memory before tiles first, first + kRun, ...; not by all CTAs at once,
    // which took each 7 us (chunk of 512 tokens, 16 tiles: 474 us, now 450)
    const int first = C::kRun - (nt > C::kRun ? id % C::kRun : 0);
    auto turn_at = [&](int j) { return j >= first && (j - first) % C::kRun == 0; };

    if (tid == 0) {
        mbar_init(&kfull, kConvWarps);
        mbar_init(&vfull, kConvWarps);
        mbar_init(&ended, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sfull[i], 1);
            mbar_init(&odone[i], 1);
            mbar_init(&pfull[i], kSoftWarps);
        }
        for (int i = 0; i < kSoftWarps; i++) {
            mbar_init(&xfull[i], 1);
            mbar_init(&xfree[i], 1);
        }
        k_top = 0;
        failed = 0;
    }
    if (tid < G) v_top[tid] = 0;
    if (tid < 4) nan_tile[tid] = 0;
    if (tid < 16) missing[tid >> 2][tid & 3] = 0;
    if (tid < 16 * G) nan_keys[0][0][tid] = make_int2(0, 0);
    mbar_fence_init();
    if (warp == kSoftWarps + kConvWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    if constexpr (CL > 1) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    griddep_launch();

    const int valid = it.tokens * (int)p.group;                 // rows of the tile: (token, head of the group)
    auto q_row = [&](int r) {                                   // its place in q (or out), in elements, given the stride
        const unsigned tok = (unsigned)r / p.group;
        return (long long)(it.row0 + it.tok0 + (int)tok);
    };
    auto head_of = [&](int r) { return (long long)(h * p.group + (unsigned)r % p.group) * HD; };

    // ---- prologue, all but the MMA warp: query operands, largest scales ----
    const int recs = nt * (kT / kKv4Rec);
    auto scan_addr = [&](int r0) -> unsigned long long {        // of this warp's next 32 records, one per lane
        const int mine = r0 + warp + lane * (kSoftWarps + kConvWarps);
        return mine < recs ? (unsigned long long)kv4_record(p.c, it.seq, (long long)t0 * kT + mine * kKv4Rec, h) : 0;
    };
    unsigned long long addr = 0;
    if (warp < kSoftWarps + kConvWarps) addr = scan_addr(0);
    if (warp < kSoftWarps + kConvWarps) {
        constexpr int LR = DC / 8 < 32 ? DC / 8 : 32;           // lanes of a row
        constexpr int RP = 32 / LR, RW = kM / (kSoftWarps + kConvWarps), NP = RW / RP;   // rows of a pass, of a warp
        constexpr int NU = NP < 4 ? NP : 4;                     // passes in flight
        const int lr = lane / LR, ch = lane % LR;
#pragma unroll 1
        for (int p0 = 0; p0 < NP; p0 += NU) {
            float x[NU][8];
            uint4 raw[NU];                                      // of 16-bit types, so that all loads are on their way at once
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const int r = warp * RW + (p0 + u) * RP + lr;
                const bool have = p0 + u < NP && r < valid;
                const long long at = have ? q_row(r) * p.q_stride + head_of(r) + rank * DC + ch * 8 : 0;
#pragma unroll
                for (int i = 0; i < 8; i++) x[u][i] = 0.0f;
                raw[u] = make_uint4(0, 0, 0, 0);
                if (HILO) {
                    if (have) Kv4Vec<float>::load((const float *)p.q + at, x[u]);
                } else if (have) raw[u] = *reinterpret_cast<const uint4 *>((const uint16_t *)p.q + at);
            }
#pragma unroll
            for (int u = 0; u < NU && !HILO; u++)
                load8(&raw[u], p.type, 0, x[u]);
#pragma unroll
            for (int u = 0; u < NU; u++) {
                if (p0 + u >= NP) break;
                const int r = warp * RW + (p0 + u) * RP + lr;
                float mx = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[u][i]));
#pragma unroll
                for (int o = 1; o < LR; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 115);
                const float up = pow2(13 - e);
                if (ch == 0) q_inv[r] = pow2(e - 13);
                // dimensions in the order in which a word's codes come out: 0, 4, 1, 5, 2, 6, 3, 7
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float a = x[u][i] * up, b = x[u][i + 4] * up;
                    hi[i] = pack_h(a, b);
                    if (HILO) {
                        const float2 f = unpack_h(hi[i]);
                        lo[i] = pack_h(a - f.x, b - f.y);
                    }
                }
                const int to = (ch >> 3) * (kM * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
                *reinterpret_cast<uint4 *>(qh + to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (HILO) *reinterpret_cast<uint4 *>(ql + to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        fence_async();
    }
    if (warp < kSoftWarps + kConvWarps) {
        // The largest scales: a warp takes every 16th record, 8 at a time in flight, K scales
        // of a token per lane in its lower half, G V scales per lane in the upper one.
        constexpr int kScan = kSoftWarps + kConvWarps, kFlight = 8;
        uint32_t km = 0;
        const bool is_v = lane >= 16;
        const int i16 = lane & 15, at_lane = 16 * HD + (is_v ? 32 * HG + rank * (32 * G) + i16 * (2 * G)
                                                              : i16 * (2 * HG) + rank * (2 * G));
        for (int r0 = 0; r0 < recs; r0 += 32 * kScan) {
            if (r0) addr = scan_addr(r0);
            const int left = (recs - r0 - warp + kScan - 1) / kScan;
            for (int k0 = 0; k0 < min(left, 32); k0 += kFlight) {
                uint32_t w[kFlight][2];
#pragma unroll
                for (int u = 0; u < kFlight; u++) {
                    const uint8_t *src = (const uint8_t *)__shfl_sync(0xffffffffu, addr, k0 + u);
                    w[u][0] = w[u][1] = 0;
                    if (!src) continue;
                    if constexpr (G == 4) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(src + at_lane);
                        w[u][0] = x.x;
                        w[u][1] = x.y;
                    } else if constexpr (G == 2) w[u][0] = *reinterpret_cast<const uint32_t *>(src + at_lane);
                    else w[u][0] = *reinterpret_cast<const uint16_t *>(src + at_lane);
                }
#pragma unroll
                for (int u = 0; u < kFlight; u++) {
                    const int key = t0 * kT + (r0 + warp + (k0 + u) * kScan) * kKv4Rec;
                    const bool inside = key >= it.see0 && key + kKv4Rec - 1 <= it.see1;
#pragma unroll
                    for (int x = 0; x < G; x++) {
                        const uint32_t a = w[u][x / 2] >> (16 * (x & 1)) & 0xffffu;
                        const int at = i16 * G + x, tok = is_v ? 2 * (at >> 2 & 3) + (at & 1) + 8 * (at >> 1 & 1) : i16;
                        if (a < 0x7f80u && (inside || (key + tok >= it.see0 && key + tok <= it.see1))) km = max(km, a);
                    }
                }
            }
        }
        // K in the lower half of the warp, V in the upper one, 16 / G lanes a group
#pragma unroll
        for (int o = 1; o < 16 / G; o <<= 1) km = max(km, __shfl_xor_sync(0xffffffffu, km, o));
        if (lane % (16 / G) == 0) atomicMax(is_v ? &v_top[i16 / (16 / G)] : &k_top, km);
    }
    __syncthreads();
    // scales times 2^up are at most 2^12; an operand is then the value times 2^(up - 17). Values
    // have a factor for each group of dimensions (columns of their own in the output).
    auto up_of = [](uint32_t top) { return top ? min(max(11 - ((int)(top >> 7) - 127), -100), 113) : 0; };
    const int ka = up_of(k_top);

    // A wait ran out: this thread waits no more, and the rows of both CTAs are NaN, whose
    // scores are made of both halves.
    bool lost = false;
    auto fail = [&]() {
        lost = true;
        failed = 1;
        if constexpr (CL > 1) remote_store(rank_addr(smem_u32(&failed), rank ^ 1), 1);
    };
    auto wait = [&](uint64_t *bar, int phase) {
        if (!lost && !mbar_wait(bar, phase & 1, nullptr, 0)) fail();
    };
    // All warps of the row tile, when every product is done and nothing is on its way between
    // the CTAs any more: from here on `failed` says what it will say.
    auto meet = [&]() {
        __syncwarp();
        if constexpr (CL > 1) cluster_sync();
        else __syncthreads();
    };

    if (warp == kSoftWarps + kConvWarps) {
        // ---- the MMAs ----
        constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(kM >> 4) << 24);       // fp16, fp16 -> fp32
        constexpr uint32_t kIdS = kIdesc | ((uint32_t)(kT >> 3) << 17), kIdO = kIdesc | ((uint32_t)(DC >> 3) << 17);
        if (lane == 0) {
            // S runs two tiles ahead of P V, so that the softmax of a tile never waits for an S
            // that stands behind its own P V. (S_{j+2} overwrites S_j: P_j says that it was read.)
            for (int j = -2; j < nt; j++) {
                if (j >= 0) {
                    const int b = j & 1;
                    wait(&vfull, j);
                    wait(&pfull[b], j >> 1);
                    tc_fence_after();
#pragma unroll
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int i = 0; i < kT / 16; i++)
                            mma_f16_ta(tmem + kColO, tmem + kColP + b * 64 + half * 32 + i * 8, umma_desc(vb, i * 32),
                                       kIdO, (j && !turn_at(j)) || half || i);
                    mma_commit(&odone[b]);
                }
                if (j + 2 < nt) {
                    wait(&kfull, j + 2);
                    tc_fence_after();
                    const uint32_t d = tmem + kColS + (j & 1) * kT;
                    // the low halves of q first: the tensor cores truncate by the size of the sum
                    // (fp32 outputs of a chunk at 16384 keys 5.0e-6 off, now 3.3e-6)
#pragma unroll
                    for (int half = 0; half < (HILO ? 2 : 1); half++)
#pragma unroll
                        for (int i = 0; i < G * 4; i++)
                            mma_f16(d, umma_desc((HILO && !half ? ql : qh) + (i >> 2) * (kM * 128), (i & 3) * 32),
                                    umma_desc(kb + (i >> 2) * (kT * 128), (i & 3) * 32), kIdS, half || i);
                    mma_commit(&sfull[j & 1]);
                }
            }
            mma_commit(&ended);                                 // no MMA is left when TMEM is freed
            if (!mbar_wait(&ended, 0, nullptr, 0)) fail();
        }
        meet();
    } else if (warp >= kSoftWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvRegs));
        // ---- conversion: this warp's record of each tile, its groups g0, g0 + 2, ... ----
        const int cw = warp - kSoftWarps, rec = cw & 3, g0 = cw >> 2;
        const bool busy = g0 < G;
        const int g = lane >> 2, t = lane & 3;
        const float kup = pow2(ka);
        float vup[NB];
#pragma unroll
        for (int n = 0; n < NB; n++) vup[n] = pow2(up_of(v_top[busy ? g0 + 2 * n : 0]));
        // the page of this warp's record of tile j (loaded an iteration before it is looked at),
        // and the record's address
        const int *table = p.c.table + (long long)it.seq * p.c.table_stride;
        auto page_of = [&](int j) -> int {
            const int slot = ((t0 + j) * kT + rec * 16) >> p.c.page_shift;
            return j < nt && slot < p.c.table_stride ? table[slot] : -1;
        };
        auto record = [&](int j, int page) -> const uint8_t * {
            if ((unsigned)page >= (unsigned)p.c.num_pages) return nullptr;
            const int in_page = ((t0 + j) * kT + rec * 16) & ((1 << p.c.page_shift) - 1);
            return p.c.pages + page * p.c.page_bytes + (long long)(((h << p.c.page_shift) + in_page) >> 4) * (17 * HD);
        };
        uint4 kc[NB], vc[NB];
        uint32_t ks[NB];                                        // scales of keys g and g + 8
        uint2 vs[NB], vn[NB];                                   // of keys 2t, 2t + 1, 2t + 8, 2t + 9; the next tile's
        auto fetch_k = [&](const uint8_t *src) {                // K codes, all scales
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const int gr = rank * G + g0 + 2 * n;
                kc[n] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
                ks[n] = 0;
                vn[n] = make_uint2(0, 0);
                if (src && busy) {
                    const uint16_t *sc = reinterpret_cast<const uint16_t *>(src + 16 * HD);
                    kc[n] = *reinterpret_cast<const uint4 *>(src + gr * 512 + lane * 16);
                    ks[n] = (uint32_t)sc[g * HG + gr] | (uint32_t)sc[(g + 8) * HG + gr] << 16;
                    vn[n] = *reinterpret_cast<const uint2 *>(sc + 16 * HG + gr * 16 + t * 4);
                }
            }
        };
        auto fetch_v = [&](const uint8_t *src) {
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const int gr = rank * G + g0 + 2 * n;
                vc[n] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
                if (src && busy) vc[n] = *reinterpret_cast<const uint4 *>(src + 8 * HD + gr * 512 + lane * 16);
            }
        };
        // K rows are keys: a word's 8 dimensions are one 16-byte chunk
        auto convert_k = [&](int j) {
            if (j > 0) wait(&sfull[(j - 1) & 1], (j - 1) >> 1);             // S_{j-1} has read the buffer
            if (busy) {
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    const uint32_t w[4] = {kc[n].x, kc[n].y, kc[n].z, kc[n].w};
                    uint8_t *tile = kb + (g0 + 2 * n) * (kT * 128);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float f = bound(__uint_as_float(i ? ks[n] & 0xffff0000u : ks[n] << 16) * kup);
                        const uint32_t s = pack_h(f, f), s16 = pack_h(f * 16.0f, f * 16.0f),
                                       off = mul_h(s, 0x84008400u);        // -2^-14 S
                        const int row = rec * 16 + g + 8 * i;
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const uint32_t x = w[2 * i + u] << 3, y = w[2 * i + u] >> 5;
                            const uint4 v4 = make_uint4(value2(x, kLoMask, s16, off), value2(x, kHiMask, s, off),
                                                        value2(y, kLoMask, s16, off), value2(y, kHiMask, s, off));
                            *reinterpret_cast<uint4 *>(tile + row * 128 + (((2 * t + u) ^ (row & 7)) << 4)) = v4;
                        }
                    }
                }
            }
            fence_async();
            __syncwarp();
            if (STARVE && blockIdx.x == 0) {
                if (p.starve == 1) return;
                if (p.starve == 2 && warp == kSoftWarps) fail();
            }
            if (lane == 0) mbar_arrive(&kfull);
        };
        // NaN among the values of tile j: remembered by key, the operand is 0
        auto find_nan = [&](int j) {
            bool bad = false;
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const uint32_t w[2] = {vn[n].x, vn[n].y};
#pragma unroll
                for (int i = 0; i < 2; i++) bad |= (w[i] & 0x7fffu) > 0x7f80u || (w[i] >> 16 & 0x7fffu) > 0x7f80u;
            }
            if (!__any_sync(0xffffffffu, bad)) return;
#pragma unroll
            for (int n = 0; n < NB; n++) {
                uint32_t keys = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t s = (i < 2 ? vn[n].x : vn[n].y) >> (16 * (i & 1)) & 0xffffu;
                    if ((s & 0x7fffu) > 0x7f80u) {
                        keys |= 1u << (2 * t + (i & 1) + 8 * (i >> 1));
                        if (i < 2) vn[n].x &= ~(0xffffu << (16 * (i & 1)));
                        else vn[n].y &= ~(0xffffu << (16 * (i & 1)));
                    }
                }
                keys = __reduce_or_sync(0xffffffffu, keys);
                if (lane == 0) {
                    nan_keys[j & 3][g0 + 2 * n][rec] = make_int2(j + 1, (int)keys);
                    nan_tile[j & 3] = j + 1;
                }
            }
        };
        // V^T rows are dimensions: a pair of keys is 4 bytes. Lane g starts with dimension
        // 8 g + g % 8, so that the lanes of a store fall into different chunks.
        auto convert_v = [&](int j) {
            if (j > 0) wait(&odone[(j - 1) & 1], (j - 1) >> 1);             // P_{j-1} V has read the buffer
            if (busy) {
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    const uint32_t rot = 4 * g;
                    const uint32_t w0 = __funnelshift_r(vc[n].x, vc[n].x, rot), w1 = __funnelshift_r(vc[n].y, vc[n].y, rot),
                                   w2 = __funnelshift_r(vc[n].z, vc[n].z, rot), w3 = __funnelshift_r(vc[n].w, vc[n].w, rot);
#pragma unroll
                    for (int pr = 0; pr < 2; pr++) {
                        const uint32_t sw = pr ? vs[n].y : vs[n].x;
                        const float f0 = bound(__uint_as_float(sw << 16) * vup[n]),
                                    f1 = bound(__uint_as_float(sw & 0xffff0000u) * vup[n]);
                        const uint32_t s = pack_h(f0, f1), s16 = pack_h(f0 * 16.0f, f1 * 16.0f),
                                       off = mul_h(s, 0x84008400u);
                        const int key = rec * 16 + 8 * pr + 2 * t;          // keys key, key + 1
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const uint32_t ab = __byte_perm(pr ? w2 : w0, pr ? w3 : w1, u ? 0x7632 : 0x5410);
                            const uint32_t x = ab << 3, y = ab >> 5;
                            const uint32_t v4[4] = {value2(x, kLoMask, s16, off), value2(x, kHiMask, s, off),
                                                    value2(y, kLoMask, s16, off), value2(y, kHiMask, s, off)};
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int d = (4 * u + i + g) & 7;          // dimension 8 g + d of the group
                                const int row = (g0 + 2 * n) * 64 + 8 * g + d;
                                *reinterpret_cast<uint32_t *>(vb + row * 128 + (((key >> 3) ^ d) << 4) +
                                                              (key & 7) * 2) = v4[i];
                            }
                        }
                    }
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&vfull);
        };
        // what the softmax has to know of tile j, before its K is passed on
        auto note = [&](int j, const uint8_t *src) {
            if (!src && lane == 0) missing[j & 3][rec] = j + 1;
            if (busy) find_nan(j);
        };
        // K is converted two tiles ahead of V, like the MMAs. In registers at the top of the
        // loop: V of tile j; K and all scales of tile j + 2; the V scales of tile j + 1.
        uint2 v1[NB];
        auto keep = [&](uint2 (&to)[NB], const uint2 (&from)[NB]) {
#pragma unroll
            for (int n = 0; n < NB; n++) to[n] = from[n];
        };
        const uint8_t *r1 = record(1, page_of(1)), *r2 = record(2, page_of(2));       // of tiles j + 1, j + 2
        int page = page_of(3);                                                        // of tile j + 3
        {
            const uint8_t *r0 = record(0, page_of(0));
            fetch_k(r0);
            fetch_v(r0);
            if (nt > 0) {
                note(0, r0);
                convert_k(0);
                keep(vs, vn);
                fetch_k(r1);
            }
            if (nt > 1) {
                note(1, r1);
                convert_k(1);
                keep(v1, vn);
                fetch_k(r2);
            }
        }
        for (int j = 0; j < nt; j++) {
            convert_v(j);
            if (j + 1 < nt) fetch_v(r1);
            keep(vs, v1);
            if (j + 2 < nt) {
                note(j + 2, r2);
                convert_k(j + 2);
                keep(v1, vn);
            }
            r1 = r2;
            r2 = record(j + 3, page);
            page = page_of(j + 4);
            if (j + 3 < nt) fetch_k(r2);
        }
        meet();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        // ---- softmax: threads (r, half) take keys 32 half .. + 31 of row r ----
        const int quad = warp & 3, half = warp >> 2, r = quad * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        const long long pos = it.pos0 + it.tok0 + (unsigned)r / p.group;
        const int cap = p.c.table_stride << p.c.page_shift;
        const int my_hi = r < valid ? (int)max(min(pos, (long long)cap - 1), -1ll) : -1;
        const int my_lo = p.window ? (int)min(max(pos - p.window + 1, 0ll), (long long)cap) : 0;
        // the softmax scale's sign goes with q; a scale of 0 still leaves -inf what it is
        const float cq = copysignf(q_inv[r] * pow2(min(17 - ka, 127)), p.scale),
                    rs = fmaxf(fabsf(p.scale) * kLog2e, 0x1p-120f);
        const uint32_t peer_x = CL > 1 ? rank_addr(smem_u32(xb), rank ^ 1) : 0;
        const uint32_t peer_full = CL > 1 ? rank_addr(smem_u32(&xfull[warp]), rank ^ 1) : 0;
        const uint32_t peer_free = CL > 1 ? rank_addr(smem_u32(&xfree[warp]), rank ^ 1) : 0;
        float m = -INFINITY, l = 0.0f;
        uint32_t nans = 0;                                      // groups with a NaN value that this row sees
        // the row's sum of the runs before this one, in the range's place among the partial
        // results (4 dimensions x rows, so that a warp's accesses are 512 bytes), for the reference m_acc
        auto sums = [&]() { return p.parts + (long long)(blockIdx.x / CL) * (kM * HD) + rank * (kM * DC) + r * 4; };
        float m_acc = -INFINITY;
        auto factor = [&]() { return m_acc == m ? 1.0f : ex2(m_acc - m); };
        // this CTA's half of S of a tile to the other CTA: on its way while the tile before
        // it is worked on
        const int x0 = (half * (kH / 4)) * kM + r;
        // The warps of the pair go on or give up together: one that is lost sends nothing more and
        // frees nothing, so that the other's waits run out too.
        auto send = [&](int j) {
            wait(&sfull[j & 1], j >> 1);
            tc_fence_after();
            if (j > 0 && !lost && !wait_cluster(&xfree[warp], (j - 1) & 1)) fail();
            if (__any_sync(0xffffffffu, lost)) {
                if (!lost) fail();
                return;
            }
#pragma unroll
            for (int c = 0; c < kH; c += 16) {
                int v[16];
                tmem_ld16(lanes + kColS + (j & 1) * kT + half * kH + c, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 4; i++)
                    remote_store4(peer_x + (uint32_t)(x0 + (c / 4 + i) * kM) * 16, __int_as_float(v[4 * i]) * cq,
                                  __int_as_float(v[4 * i + 1]) * cq, __int_as_float(v[4 * i + 2]) * cq,
                                  __int_as_float(v[4 * i + 3]) * cq, peer_full);
            }
            if (lane == 0) mbar_arrive_expect_tx(&xfull[warp], C::kX / kSoftWarps);
        };
        if (CL > 1 && nt > 0) send(0);
        for (int j = 0; j < nt; j++) {
            const int b = j & 1;
            float s[kH];
            if constexpr (CL == 1) {
                wait(&sfull[b], j >> 1);
                tc_fence_after();
            } else if (!lost && !wait_cluster(&xfull[warp], j & 1)) fail();
            {
                int v[kH];
                tmem_ld32(lanes + kColS + b * kT + half * kH, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < kH / 4; i++) {
                    // the halves of S: each CTA adds the other's to its own. Both sums are the
                    // same bits: the product with a power of two is exact.
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if constexpr (CL > 1) x = xb[x0 + i * kM];
                    s[4 * i] = fmaf(__int_as_float(v[4 * i]), cq, x.x);
                    s[4 * i + 1] = fmaf(__int_as_float(v[4 * i + 1]), cq, x.y);
                    s[4 * i + 2] = fmaf(__int_as_float(v[4 * i + 2]), cq, x.z);
                    s[4 * i + 3] = fmaf(__int_as_float(v[4 * i + 3]), cq, x.w);
                }
            }
            if constexpr (CL > 1) {
                if (__any_sync(0xffffffffu, lost)) lost = true;
                else if (lane == 0) remote_arrive(peer_free);
            }
            const int key0 = (t0 + j) * kT + half * kH;
            const bool gap0 = missing[j & 3][2 * half] == j + 1, gap1 = missing[j & 3][2 * half + 1] == j + 1;
            if (gap0 || gap1 || key0 < it.all0 || key0 + kH - 1 > it.all1) {
#pragma unroll
                for (int i = 0; i < kH; i++)
                    if (key0 + i < my_lo || key0 + i > my_hi || (i < 16 ? gap0 : gap1)) s[i] = -INFINITY;
            }
            if (nan_tile[j & 3] == j + 1) {
                for (int gr = 0; gr < G; gr++)
                    for (int rec = 2 * half; rec < 2 * half + 2; rec++) {
                        const int2 w = nan_keys[j & 3][gr][rec];
                        if (w.x == j + 1)
                            for (int i = 0; i < 16; i++) {
                                const int key = (t0 + j) * kT + rec * 16 + i;
                                if ((w.y >> i & 1) && key >= my_lo && key <= my_hi) nans |= 1u << gr;
                            }
                    }
            }
            float mx4[4];
#pragma unroll
            for (int i = 0; i < 4; i++) mx4[i] = s[i];
#pragma unroll
            for (int i = 4; i < kH; i++) mx4[i & 3] = fmaxf(mx4[i & 3], s[i]);
            float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            // the row's other half; the buffers alternate
            pair[b][half][r] = mx;
            bar_sync(1 + quad, 64);
            mx = fmaxf(mx, pair[b][half ^ 1][r]) * rs;
            const bool grow = mx > m + kSlack, turn = turn_at(j);
            if (turn) {                                         // the run up to tile j - 1 is complete
                wait(&odone[b ^ 1], (j - 1) >> 1);
                tc_fence_after();
                const float f = factor();
                float *acc = sums();
                // Nothing but this thread touches its sums, so additions in memory have one
                // order. The reference rarely moves once a few tiles are done.
                const bool same = __all_sync(0xffffffffu, f == 1.0f);
#pragma unroll 1
                for (int c = half * (DC / 2); c < (half + 1) * (DC / 2); c += 32) {
                    int v[32];
                    tmem_ld32(lanes + kColO + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        float4 *to = reinterpret_cast<float4 *>(acc + (c + x) * kM);
                        float4 y = make_float4(__int_as_float(v[x]), __int_as_float(v[x + 1]), __int_as_float(v[x + 2]),
                                               __int_as_float(v[x + 3]));
                        if (j == first) __stcg(to, y);
                        else if (same) red_add4(&to->x, y.x, y.y, y.z, y.w);
                        else {
                            const float4 z = __ldcg(to);
                            __stcg(to, make_float4(fmaf(z.x, f, y.x), fmaf(z.y, f, y.y), fmaf(z.z, f, y.z), fmaf(z.w, f, y.w)));
                        }
                    }
                }
                m_acc = m;
            }
            if (__any_sync(0xffffffffu, grow)) {                // the same in both warps of the rows
                const float mn = grow ? mx + kHead : m, al = mn == m ? 1.0f : ex2(m - mn);
                m = mn;
                l *= al;
                if (j > 0 && !turn) {                           // (after a turn the next P V starts O anew)
                    wait(&odone[b ^ 1], (j - 1) >> 1);          // O is complete up to tile j - 1
                    tc_fence_after();
                    for (int c = half * (DC / 2); c < (half + 1) * (DC / 2); c += 32) {
                        int v[32];
                        tmem_ld32(lanes + kColO + c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; x++) v[x] = __float_as_int(__int_as_float(v[x]) * al);
                        tmem_st32(lanes + kColO + c, v);
                    }
                    tmem_wait_st();
                }
            }
            if (CL > 1 && j + 1 < nt) send(j + 1);
            const float mref = (m == -INFINITY ? 0.0f : m) - kUp;
            uint32_t ph[kH / 2], pl[kH / 2];
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kH / 2; i++) {
                const float a = ex2(fmaf(s[2 * i], rs, -mref)), c = ex2(fmaf(s[2 * i + 1], rs, -mref));
                sum[i & 3] += a + c;
                ph[i] = pack_h(a, c);
                const float2 f = unpack_h(ph[i]);
                pl[i] = pack_h(a - f.x, c - f.y);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (j > 1) wait(&odone[b], (j - 2) >> 1);           // P V of j - 2 has read this P
            tmem_st16(lanes + kColP + b * 64 + half * 16, ph);
            tmem_st16(lanes + kColP + b * 64 + 32 + half * 16, pl);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pfull[b]);
        }
        if (nt > 0) wait(&odone[(nt - 1) & 1], (nt - 1) >> 1);
        // what the other CTA may have sent is still on its way: whichever phase is not complete
        if (CL > 1 && lost)
            for (int i = 0; i < 2; i++) wait_cluster(&xfull[warp], i);
        meet();
        tc_fence_after();
        // ---- output: each thread of a row half of the dimensions ----
        pair[0][half][r] = l;
        pair[1][half][r] = __uint_as_float(failed ? 0xffffffffu : nans);
        bar_sync(1 + quad, 64);
        l += pair[0][half ^ 1][r];
        nans |= __float_as_uint(pair[1][half][r]) | __float_as_uint(pair[1][half ^ 1][r]);
        const bool part = p.splits > 1;
        const long long item = blockIdx.x / CL;
        float *acc = sums();
        const float f = factor();
        const float inv = part ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        if (part && rank == 0 && half == 0) {
            p.stats[item * (2 * kM) + r] = m;
            p.stats[item * (2 * kM) + kM + r] = l;
        }
#pragma unroll 1
        for (int c = half * (DC / 2); c < (half + 1) * (DC / 2); c += 32) {
            int v[32];
            if (nt > 0) {
                tmem_ld32(lanes + kColO + c, v);
                tmem_wait_ld();
            } else {
#pragma unroll
                for (int x = 0; x < 32; x++) v[x] = 0;
            }
            if (nt > first) {
#pragma unroll
                for (int x = 0; x < 32; x += 4) {
                    const float4 y = __ldcg(reinterpret_cast<const float4 *>(acc + (c + x) * kM));
                    v[x] = __float_as_int(fmaf(y.x, f, __int_as_float(v[x])));
                    v[x + 1] = __float_as_int(fmaf(y.y, f, __int_as_float(v[x + 1])));
                    v[x + 2] = __float_as_int(fmaf(y.z, f, __int_as_float(v[x + 2])));
                    v[x + 3] = __float_as_int(fmaf(y.w, f, __int_as_float(v[x + 3])));
                }
            }
            const bool bad = nans >> (c / kKv4Group) & 1;
            const float fac = pow2(min(17 - up_of(v_top[c / kKv4Group]), 127)) * inv;
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = bad ? NAN : __int_as_float(v[x + i]) * fac;
                if (part) {
                    *reinterpret_cast<float4 *>(acc + (c + x) * kM) = make_float4(y[0], y[1], y[2], y[3]);
                    *reinterpret_cast<float4 *>(acc + (c + x + 4) * kM) = make_float4(y[4], y[5], y[6], y[7]);
                }
                else if (r < valid)
                    store8(p.out, p.type, q_row(r) * p.out_stride + head_of(r) + rank * DC + c + x, y);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kSoftWarps + kConvWarps) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Joins the key ranges of a row tile: block (slot x kv head, 8 rows).
template <int HD>
__global__ void __launch_bounds__(kJoinThreads) k_kv4_prompt_join(const __grid_constant__ PromptP p) {
    __shared__ float f[32][8], inv[8];
    const int tid = threadIdx.x, r0 = blockIdx.y * 8;
    const int slot = p.slots - 1 - blockIdx.x / p.c.kv_heads, h = blockIdx.x % p.c.kv_heads;      // as the kernel before
    griddep_wait();
    Item it;
    if (!find_item(p, slot, it)) return;
    const int valid = it.tokens * (int)p.group;
    if (r0 >= valid) return;
    const long long item = (long long)blockIdx.x * p.splits;
    if (tid < 8) {
        const float *st = p.stats + item * (2 * kM) + r0 + tid;
        float m = -INFINITY, l = 0.0f;
        for (int s = 0; s < p.splits; s++) m = fmaxf(m, st[s * (2 * kM)]);
        const float ref = m == -INFINITY ? 0.0f : m;
        for (int s = 0; s < p.splits; s++) {
            const float x = ex2(st[s * (2 * kM)] - ref);
            f[s][tid] = x;
            l = fmaf(x, st[s * (2 * kM) + kM], l);
        }
        inv[tid] = l == 0.0f ? 0.0f : 1.0f / l;
    }
    __syncthreads();
    for (int i = tid; i < HD; i += kJoinThreads) {              // 8 rows of HD / 8 pieces
        const int r = i % 8, d = i / 8 * 8;
        const float *from = p.parts + item * (kM * HD) + (d * kM + (r0 + r) * 4);
        float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int s = 0; s < p.splits; s++) {
            __align__(16) float y[8];
            *reinterpret_cast<float4 *>(y) = *reinterpret_cast<const float4 *>(from + s * (kM * HD));
            *reinterpret_cast<float4 *>(y + 4) = *reinterpret_cast<const float4 *>(from + s * (kM * HD) + 4 * kM);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = fmaf(f[s][r], y[j], x[j]);
        }
        if (r0 + r < valid) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= inv[r];
            const unsigned tok = (unsigned)(r0 + r) / p.group;
            store8(p.out, p.type,
                   (long long)(it.row0 + it.tok0 + (int)tok) * p.out_stride +
                       (long long)(h * p.group + (unsigned)(r0 + r) % p.group) * HD + d, x);
        }
    }
}

// Key ranges of a row tile that sees `tiles` key tiles, by the time of the rounds that
// the row tiles then take: a key tile costs 1, a range (its queries and scales) about 3,
// its partial result in memory hd / 20000. At most 32, and four rounds: more would not fill the GPU better, and the
// partial outputs would grow.
int ranges(const Kv4View &c, long long items, long long tiles) {
    const long long room = kSms / (c.hd > 256 ? 2 : 1);
    double best = 0.0;
    int n = 1;
    for (int s = 1; s <= 32 && s <= tiles && (s == 1 || items * s <= 4 * room); s++) {
        const double cost = (double)((items * s + room - 1) / room) * ((double)tiles / s + 3.0) +
                            (s > 1 ? (double)(items * s) * c.hd / 20000.0 : 0.0);
        if (s == 1 || cost < 0.97 * best) {
            best = cost;
            n = s;
        }
    }
    return n;
}
// (The window can only make the ranges fewer: the workspace is sized without it.)
void plan(const Kv4View &c, unsigned group, int window, int *tokens, int *slots, int *splits) {
    *tokens = kM / (int)group;
    *slots = c.rows / *tokens + c.n;
    const long long items = (long long)((c.rows + *tokens - 1) / *tokens) * c.kv_heads,
                    tiles = (((long long)c.table_stride << c.page_shift) + kT - 1) / kT;
    *splits = ranges(c, items, tiles);
    if (window) {
        const long long seen = ((long long)window + *tokens - 1) / kT + 2;
        if (seen < tiles) {
            const int s = ranges(c, items, seen);
            if (s < *splits) *splits = s;
        }
    }
}

template <int HD, bool HILO, bool STARVE = false>
cudaError_t launch_prompt(const PromptP &p, cudaStream_t st) {
    using C = Cfg<HD, HILO>;
    constexpr auto kernel = k_kv4_prompt<HD, HILO, STARVE>;
    cudaError_t e = g4_smem_optin((const void *)kernel, C::kSmem);
    if (e != cudaSuccess) return e;
    static std::atomic<bool> fits{false};                       // a build with fewer registers would wait for more
    if (!fits) {
        cudaFuncAttributes a;
        e = cudaFuncGetAttributes(&a, (const void *)kernel);
        if (e != cudaSuccess) return e;
        if (a.numRegs < kRegs) return cudaErrorLaunchOutOfResources;
        fits = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.slots * p.c.kv_heads * p.splits * C::kCl);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = C::kCl;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C::kCl > 1 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return g4_launch(k_kv4_prompt_join<HD>, dim3((unsigned)p.slots * p.c.kv_heads, kM / 8), dim3(kJoinThreads), 0, st,
                     true, p);
}

template <int HD>
cudaError_t launch_hd(const PromptP &p, cudaStream_t st) {
    if constexpr (HD >= 256)
        if (p.starve) return p.type == G4_TYPE_F32 ? launch_prompt<HD, true, true>(p, st) : cudaErrorNotSupported;
    if (p.starve) return cudaErrorNotSupported;
    return p.type == G4_TYPE_F32 ? launch_prompt<HD, true>(p, st) : launch_prompt<HD, false>(p, st);
}

}  // namespace

// Bytes that any call of at most c.rows rows, c.n sequences and c.table_stride pages takes, of
// those that come here: plan() gives fewer rows more key ranges of a tile (bounded by 4 room /
// items in ranges()), so every number of row tiles that may be cut is looked at.
size_t kv4_prompt_ws(const Kv4View &c, int type, int q_heads) {
    const int group = q_heads / c.kv_heads, tokens = kM / group;
    const long long room = kSms / (c.hd > 256 ? 2 : 1), all = (c.rows + tokens - 1) / tokens,
                    tiles = (((long long)c.table_stride << c.page_shift) + kT - 1) / kT;
    const int run = type == G4_TYPE_F32 ? Cfg<64, true>::kRun : Cfg<64, false>::kRun;
    long long most = 0;
    for (long long t = 1; t <= all; t++) {
        long long splits = 4 * room / (t * c.kv_heads);
        splits = std::min(std::min(splits, 32ll), tiles);
        if (splits < 2) {
            t = all;                                            // not cut: the most rows need most
            splits = tiles > run ? 1 : 0;                       // of tiles, to be summed up
        }
        Kv4View v = c;                                          // the most sequences that make it many rows
        v.rows = (int)std::min<long long>(t * tokens, c.rows);
        v.n = (int)std::min<long long>(c.n, (long long)v.rows * group / kManyRows);
        if (v.n > 0 && !many_rows(v, q_heads)) v.n = (int)std::min<long long>(c.n, (long long)v.rows * group / kManyRowsAlone);
        if (v.n > 0) most = std::max(most, (v.rows / tokens + v.n) * splits);
    }
    return (size_t)most * c.kv_heads * kM * (c.hd + 2) * sizeof(float);
}

cudaError_t kv4_launch_prompt(const Kv4View &c, int type, int q_heads, const void *q, long long q_stride, void *out,
                              long long out_stride, float scale, int window, void *ws, int starve,
                              cudaStream_t st) {
    PromptP p;
    p.c = c;
    p.type = type;
    p.group = q_heads / c.kv_heads;
    plan(c, p.group, window, &p.tokens, &p.slots, &p.splits);
    p.q = q;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.scale = scale;
    p.window = window;
    p.starve = starve;
    p.parts = (float *)ws;
    p.stats = p.parts + (size_t)p.slots * c.kv_heads * p.splits * kM * c.hd;
    if (c.hd == 64) return launch_hd<64>(p, st);
    if (c.hd == 128) return launch_hd<128>(p, st);
    if (c.hd == 256) return launch_hd<256>(p, st);
    return launch_hd<512>(p, st);
}
