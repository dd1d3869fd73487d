// neon_kv8_prompt.cu -- attention over the 8-bit KV cache for many query rows
// (prompts), on tcgen05 with the sums in tensor memory.
//
// A CTA takes a unit of query rows of one KV head (MT tiles of 128 rows: row r
// is query head r % group of token r / group, so all heads of a group share
// the keys' tiles) and a share of the keys, in tiles of KT:
//
//   S = Q K^T    both operands in shared memory: Q as fp16 (fp32 queries as
//                hi + lo terms, two products into one sum), K's codes as fp16
//   P            one thread per row: t = s * (row factor * block scale), lazy
//                running maximum, p = 2^(t - m), split into hi + lo, written
//                over S in tensor memory
//   O += P V     P from tensor memory (two products into one sum), V's codes
//                as fp16 in shared memory
//
// Codes are exact in fp16, so a tile of codes is half the traffic of a 16-bit
// cache and costs a conversion (two permutes and a subtraction for four
// codes), which six warps do once for all MT tiles. A warp per query tile issues
// its products; one tile's softmax runs under the other's products.
//
// P has two terms in the types of 16 bits too: one, p to 2^-11 of itself, would
// take 345 us for the bf16 prompt below, but an output far below its values then
// shows it, and an fp16 output's error is 1.4 times its own rounding's.
//
// 4096 tokens of 64 / 8 heads x 128 from an empty cache take 388 us in bf16, 2048
// in fp32 179: 1.06 PFLOP/s of products in bf16, the second of P counted. No unit
// is full: what bounds it is the chain
// score product, read, softmax, write, output product of a row tile, of which
// tensor memory holds two, and about a fifth of a CTA's time in its queries'
// conversion before and the outputs after it. Reading the next tile's scores
// early, into registers dealt out again for it, took 419 us where this order
// took 369 (with one term of P).
//
// The maximum is lazy: m only moves, and O is only rescaled, when a row's p
// would sum to more than 2^8 in a tile (the result does not depend on m), so p
// is at most 2^8; with V's scale relative to a reference that is kept within a
// factor of 4 (vr), and 2^5, p times those stays below fp16's 65504, and its
// lo term has bits down to 2^-30 of a row's largest.
#include "neon_kv8_attn.cuh"

#include <algorithm>
#include <type_traits>

namespace longctx {
namespace {

// Warps 0-7 softmax, 8-13 conversion, 14 and 15 the products, one per query tile. The launch's 512 x 128
// registers are dealt out again by warpgroup: a softmax thread holds 64 scores, their P and its sums.
constexpr int kSoftWarps = 8, kConvWarps = 6, kMmaWarp = 14;
constexpr int kThreads = 512;
constexpr int kLaunchRegs = 128, kSoftRegs = 168, kOtherRegs = 88;
static_assert(2 * kSoftRegs + 2 * kOtherRegs <= 4 * kLaunchRegs, "register split");
constexpr int kTileShift = 6, kTileKeys = 1 << kTileShift;
constexpr float kMostP = 256.f;  // 2^8: how far p may exceed 1
constexpr float kPScale = 32.f;  // 2^5

// ---- tcgen05 ----

__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// d[tmem] (+)= a b, fp16 operands, fp32 sums: a from shared memory, or from tensor memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t a) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a));
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&r)[16], uint32_t a) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(a));
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand of 128-byte-swizzled panels [rows][64 halves]: groups of eight rows are 1024
// bytes apart; `lead` is the distance of the panels (used when the panels run along M or N). The low
// word has the address (in 16 bytes) and lead, the high word is the same for all.
__device__ __forceinline__ uint32_t operand_lo(uint32_t addr, uint32_t lead) {
    return (addr & 0x3ffff) >> 4 | ((lead >> 4) & 0x3fff) << 16;
}
__device__ __forceinline__ uint64_t operand_of(uint32_t lo) {
    return (uint64_t)(1024 >> 4 | 1u << 14 | 2u << 29) << 32 | lo;
}
// The same value in every lane, and known to be.
template <typename T>
__device__ __forceinline__ T uniform(T v) { return __shfl_sync(0xffffffffu, v, 0); }
// One lane of a converged warp, always the same one.
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}
// fp16 x fp16 -> fp32, M = 128; b_mn: B's rows run along the summed dimension
__device__ __forceinline__ uint32_t instr(int n, bool b_mn) {
    return 1u << 4 | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}

// ---- waits that end: after 2 s, or once another role has given up ----
__device__ __forceinline__ bool wait_or(uint64_t* bar, uint32_t parity, volatile int* dead, unsigned* err) {
    if (bar_try(bar, parity)) return true;
    uint64_t t0, t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    for (;;) {
        if (bar_try(bar, parity)) return true;
        if (*dead) return false;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
        if (t - t0 > 2000000000ull) {
            atomicOr(err, kErrWait);
            *dead = 1;
            return false;
        }
    }
}

// A warp puts 32 query rows of a tile into shared memory as the products read them: [TERMS][panels of
// 64 values][128 rows][64] fp16, swizzled, row r times 2^e (its largest value near 2^7) and the sign of
// the scale. Returns each lane's factor |scale| log2(e) 2^-e of row row0 + lane, 0 beyond the last row.
// A lane has eight values, one 16-byte piece, of one of R rows at a time. (This code runs once per CTA, from
// a cold instruction cache: little of it, loads first, and one step of the largest values for all rows of a batch.
// Batches of twice the rows measured 390 us against 344 on a bf16 prompt with one term of P, of half the rows 348; an
// fp32 prompt took 190 and 180 against 172.)
template <int PANELS, int TERMS, typename T>
__device__ __forceinline__ float put_queries(const AttnArgs& a, int kvh, int r0, int row0, unsigned char* tile) {
    const int hd = (int)a.c.head_dim, rows = a.n * a.group, lane = threadIdx.x & 31;
    constexpr int LPR = PANELS == 1 ? 8 : PANELS == 2 ? 16 : 32, R = 32 / LPR;  // lanes of a row, rows at a time
    constexpr int U = TERMS == 1 ? 8 : 4;                                       // of those in flight
    constexpr int Q = sizeof(T) / 2;                                            // 16-byte loads of a lane
    const bool vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.qs * sizeof(T)) % 16 == 0;
    const float sign = a.scale < 0.f ? -1.f : 1.f, size = fabsf(a.scale);
    const int d = lane % LPR * 8, sub = lane / LPR;
    // token and head of the warp's first row; those of the next 32 by a product (below 2^7 rows: exact)
    const int tok0 = (r0 + row0) / a.group, head0 = r0 + row0 - tok0 * a.group;
    const unsigned magic = 65536u / (unsigned)a.group + 1u;
    float mine = 0.f;
#pragma unroll 1
    for (int i = 0; i < 32; i += R * U) {
        union { uint4 v[Q]; T t[8]; } w[U];  // the loads alone first: all of them in flight before a value is used
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = i + u * R + sub;
            const int up = (int)(((unsigned)(head0 + k) * magic) >> 16);
            const T* q = (const T*)a.q + (long long)(tok0 + up) * a.qs + (long long)(kvh * a.group + head0 + k - up * a.group) * hd + d;
            const bool on = d < hd && r0 + row0 + k < rows;
#pragma unroll
            for (int e = 0; e < Q; ++e) w[u].v[e] = make_uint4(0, 0, 0, 0);
            if (vec) {
                if (on)
#pragma unroll
                    for (int e = 0; e < Q; ++e) w[u].v[e] = reinterpret_cast<const uint4*>(q)[e];
            } else if (on) {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[u].t[e] = q[e];
            }
        }
        float most[U];  // the rows' largest values, each step for all rows: their latencies side by side
#pragma unroll
        for (int u = 0; u < U; ++u) {
            most[u] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) most[u] = fmaxf(most[u], fabsf(to_f(w[u].t[e])));
        }
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1)
#pragma unroll
            for (int u = 0; u < U; ++u) most[u] = fmaxf(most[u], __shfl_xor_sync(0xffffffffu, most[u], o));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = to_f(w[u].t[e]);
            const unsigned top = __float_as_uint(most[u]) >> 23;
            const int e2 = top >= 255u ? 0 : min(120, 134 - (int)top);
            const float f = pow2(e2) * sign;
            if (d < PANELS * 64) {
                uint4 hi, lo;
                split2(x[0] * f, x[1] * f, hi.x, lo.x);
                split2(x[2] * f, x[3] * f, hi.y, lo.y);
                split2(x[4] * f, x[5] * f, hi.z, lo.z);
                split2(x[6] * f, x[7] * f, hi.w, lo.w);
                // piece (d % 64) / 8 of the row moves to piece ^ (row % 8)
                const int row = row0 + i + u * R + sub;
                const int at = (d >> 6) * 16384 + row * 128 + (((d & 63) >> 3 ^ (row & 7)) << 4);
                *reinterpret_cast<uint4*>(tile + at) = hi;
                if (TERMS == 2) *reinterpret_cast<uint4*>(tile + PANELS * 16384 + at) = lo;
            }
            // lane k takes the factor of row k
            const float got = __shfl_sync(0xffffffffu, size * pow2(-e2), lane % R * LPR);
            if (lane / R * R == i + u * R && r0 + row0 + lane < rows) mine = got;
        }
    }
    return mine;
}

// 16 values of a thread's row, in whole 32-byte sectors where the address allows.
template <typename T>
__device__ __forceinline__ void store16(T* d, const T (&w)[16]) {
    constexpr int N = sizeof(T) * 4;  // words
    uint32_t x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (sizeof(T) == 4) x[i] = __float_as_uint(w[i]);
        else x[i] = (uint32_t)*reinterpret_cast<const uint16_t*>(&w[2 * i]) | (uint32_t)*reinterpret_cast<const uint16_t*>(&w[2 * i + 1]) << 16;
    }
    if ((reinterpret_cast<uintptr_t>(d) & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 8)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint32_t*>(d) + i),
                         "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]),
                         "r"(x[i + 7])
                         : "memory");
    } else if ((reinterpret_cast<uintptr_t>(d) & 15) == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) reinterpret_cast<uint4*>(d)[i / 4] = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) d[i] = w[i];
    }
}

// Where 16 codes (values 16 c .. of row r) begin in a swizzled tile of `height` rows, and putting them
// there: eight of them as halves fill one 16-byte piece, the other eight the neighbouring one.
__device__ __forceinline__ int put_at(int height, int r, int c) {
    return (c >> 2) * (height * 128) + r * 128 + (((2 * (c & 3)) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void put_codes(unsigned char* tile, int at, uint4 w) {
    const uint32_t u[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
    *reinterpret_cast<uint4*>(tile + at) = make_uint4(codes_lo(u[0]), codes_hi(u[0]), codes_lo(u[1]), codes_hi(u[1]));
    *reinterpret_cast<uint4*>(tile + (at ^ 16)) = make_uint4(codes_lo(u[2]), codes_hi(u[2]), codes_lo(u[3]), codes_hi(u[3]));
}

// ---------------------------------------------------------------------------
// The main kernel
// ---------------------------------------------------------------------------
template <int PANELS, int TERMS>
struct Shape {
    static constexpr int MT = PANELS <= 2 ? 2 : 1;       // query tiles of 128 rows
    static constexpr int KT = kTileKeys;                 // keys of a tile
    static constexpr int QTile = TERMS * PANELS * 16384;
    static constexpr int Stage = PANELS * KT * 128;
    static constexpr int fits(int st) { return MT * QTile + 2 * st * Stage + 1024 + 512 <= 232448; }
    static constexpr int ST = fits(4) ? 4 : fits(2) ? 2 : 1;  // tiles of K, and of V, held at once
    static constexpr int Ahead = ST > 1 ? 2 : 1;              // tiles that the scores are ahead of the outputs
    static constexpr int Smem = MT * QTile + 2 * ST * Stage + 1024 + 512;
    static constexpr int SCols = 2 * KT, OCols = PANELS * 64;  // two buffers of S
    static_assert(MT * (SCols + OCols) <= 512, "tensor memory");
    static_assert(Smem <= 232448, "shared memory");
};

struct Bars {
    uint64_t q, k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2][2], p_full[2][2], o_done[2], o_full[2], drain[2];
    uint32_t tmem;
    int dead;
};
static_assert(sizeof(Bars) <= 512, "barriers");

template <int PANELS, typename T, int TERMS = sizeof(T) == 4 ? 2 : 1>
__global__ void __launch_bounds__(kThreads, 1) kv8_prompt_kernel(const __grid_constant__ AttnArgs a, int tiles128) {
    using S = Shape<PANELS, TERMS>;
    constexpr int MT = S::MT, KT = S::KT, ST = S::ST, NB = KT / 32;
    // What a tile's products cut off of their sums, as a part of the sum: some 0.4 ulps (an ulp is 0.72 * 2^-23 of a
    // number in the mean) in each of KT / 16 steps of two terms. Measured over 950 keys: an fp32 output of equal values
    // is 4.6e-6 short (0.88 ulps a step), one of values from 0.5 to 1.5 3.1e-6; with this added back 2.3e-6 and 8e-7,
    // and one of values of either sign is 5.7e-7 off where it was 9.7e-7 (0.5 ulps: 1.7e-6, 2e-7 and 7.5e-7).
    constexpr float kCut = 2 * (KT / 16) * 0.4f * 0.72f / 8388608.f;
    static_assert(NB == 2, "two blocks a tile");
    constexpr int kChain = (TERMS == 2 ? kChainKeys : kChainKeys16) / KT;  // tiles whose outputs are summed in tensor memory
    extern __shared__ unsigned char raw[];
    unsigned char* smem = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    unsigned char *qs = smem, *ks = qs + MT * S::QTile, *vs = ks + ST * S::Stage;
    Bars* bar = reinterpret_cast<Bars*>(vs + ST * S::Stage);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hd = (int)a.c.head_dim, cap = (int)a.c.capacity, H = (int)a.c.n_kv_head, rows = a.n * a.group;
    // the units with the most keys first
    const int units = (rows + 128 * MT - 1) / (128 * MT);
    const int kvh = blockIdx.x % H, split = blockIdx.x / H % a.nsplit, unit = units - 1 - blockIdx.x / (H * a.nsplit);
    if (warp == kMmaWarp) {
        if (lane == 0) {
            bar_init(&bar->q, 4 * MT);
            for (int i = 0; i < 4; ++i) {
                bar_init(&bar->k_full[i], kConvWarps);
                bar_init(&bar->k_empty[i], MT);
                bar_init(&bar->v_full[i], kConvWarps);
                bar_init(&bar->v_empty[i], MT);
                bar_init(&bar->s_full[i >> 1][i & 1], 1);
                bar_init(&bar->p_full[i >> 1][i & 1], 4);
            }
            for (int i = 0; i < 2; ++i) {
                bar_init(&bar->o_done[i], 1);
                bar_init(&bar->o_full[i], 1);
            }
            bar_init(&bar->drain[0], 1);
            bar_init(&bar->drain[1], 1);
            bar->dead = 0;
            bar_init_fence();
        }
        __syncwarp();
        tmem_alloc(&bar->tmem, 512);
        tc_before();
    }
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    tc_after();
    const uint32_t tmem = bar->tmem;

    const int past = *a.c.past;
    const Shares sh = shares_of(a, past, unit);
    const int j0 = min(split * sh.per, sh.tiles), j1 = min(j0 + sh.per, sh.tiles);
    // the key tiles of each query tile within the share
    int nt[MT];
    int most = 0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int first = (unit * MT + m) * 128;
        const int keys = first < rows ? keys_of(past, min(first + 127, rows - 1) / a.group, cap) : 0;
        nt[m] = max(0, min(j1, (keys + KT - 1) / KT) - j0);
        most = max(most, nt[m]);
    }

    if (warp < kSoftWarps) {
        // ---- softmax: one thread per row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        const int m = warp >> 2;
        const int r0 = (unit * MT + m) * 128, rr = r0 + (warp & 3) * 32 + lane;
        if (m < MT && (sh.has(split))) {
            const bool on = rr < rows;
            const int limit = on ? keys_of(past, rr / a.group, cap) : 0;
            const float factor = put_queries<PANELS, TERMS, T>(a, kvh, r0, (warp & 3) * 32, qs + m * S::QTile);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&bar->q);
            if (a.weight && split == 0) a.qfactor[(size_t)kvh * tiles128 * 128 + rr] = factor;
            const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's lanes: 32 (warp % 4) ..
            const uint32_t st = tmem + lanes + m * S::SCols, ot = tmem + lanes + MT * S::SCols + m * S::OCols;
            const float* ksc = a.c.k_scale + (size_t)kvh * (cap >> 5);
            const float* vsc = a.c.v_scale + (size_t)kvh * (cap >> 5);
            // the keys that every row of the warp sees
            const int all = __reduce_min_sync(0xffffffffu, limit);
            float mref = -INFINITY, l = 0.f, vref = 0.f;
            float lw = 0.f, cut = 0.f;  // fp32: a chain's sum of p's terms, and what the products cut off of it
            float held = 1.f;          // what the chains that were put by are to be multiplied with
            // those chains' sums: [32 rows][share][four columns][row][4], a warp's in whole lines
            float4* sums = a.sums + (((size_t)kvh * units * (4 * MT) + (r0 >> 5) + (warp & 3)) * a.nsplit + split) * (size_t)hd * 8 + lane;
            bool alive = true;
            float nk[NB], nv[NB];  // the scales of the next tile's blocks (a load each: quicker here than shuffles)
            auto scales = [&](int j) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int blk = min(j * NB + b, (cap >> 5) - 1);  // (past the end: of hidden keys)
                    nk[b] = ksc[blk];  // (not by the read-only path: an append that wrote them may end after this launch began)
                    nv[b] = vsc[blk];
                }
            };
            const int n = m == 0 ? nt[0] : nt[MT - 1];
            if (n) scales(j0);
            // m, and the reference of V's scales, move to what tile i needs: its largest score, and its largest
            // scale if that is above four times the reference; O and l follow.
            auto move = [&](int i, const float (&kf)[NB], float vmax) {
                const int seen = limit - (j0 + i) * KT;
                float mt = -INFINITY;
#pragma unroll 1
                for (int b = 0; b < NB; ++b) {
                    uint32_t r[32];
                    tmem_ld32(r, st + (i & 1) * KT + 32 * b);
                    tmem_wait_ld();
                    const int c = seen - 32 * b;
                    float x = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (e < c) x = fmaxf(x, __uint_as_float(r[e]));
                    if (c > 0) mt = fmaxf(mt, x * (b ? kf[NB - 1] : kf[0]));
                }
                const float mnew = fmaxf(mt, mref), vtop = vmax > 4.f * vref ? vmax : vref;
                const float fl = mref == -INFINITY ? 0.f : ex2(mref - mnew);
                const float f = vtop > 0.f ? fl * (vref / vtop) : fl;
                // O once the tile before has been added: of the outputs, i - 1 or i have ended here (the scores of
                // tile i come after output i - 2, output i needs this tile's P), so the parity is clear
                if (i % kChain && __any_sync(0xffffffffu, f != 1.f)) {
                    alive = __all_sync(0xffffffffu, wait_or(&bar->o_done[m], (uint32_t)(i - 1) & 1, &bar->dead, a.err));
                    tc_after();
#pragma unroll 1
                    for (int c = 0; c < hd; c += 16) {
                        uint32_t o[16];
                        tmem_ld16(o, ot + c);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st16(ot + c, o);
                    }
                }
                l *= fl;
                lw *= f;
                cut *= f;
                held *= f;
                mref = mnew;
                vref = vtop;
            };
            // The products cut each of their sums off towards zero, so that what came early in a long sum fades (see
            // kChainKeys). So before every kChain-th tile the outputs so far are put by, added up in fp32 in the
            // workspace, and the products begin a new sum; at the end what was put by is added to the last one.
            auto put_by = [&](int i, bool end) {
                float4 by[8];
                auto fetch = [&](int c) {  // 32 columns of what was put by before
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        by[e] = i > kChain && c + 4 * e < hd ? sums[(c + 4 * e) * 8] : make_float4(0.f, 0.f, 0.f, 0.f);
                };
                fetch(0);
                const float fix = TERMS == 2 && lw != 0.f ? 1.f + cut / lw : 1.f;
                if (!end) alive = __all_sync(0xffffffffu, wait_or(&bar->o_done[m], (uint32_t)(i - 1) & 1, &bar->dead, a.err));
                tc_after();
#pragma unroll 1
                for (int c = 0; c < hd; c += 32) {
                    if (c) fetch(c);
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        if (c + 16 * b >= hd) break;
                        uint32_t o[16];
                        tmem_ld16(o, ot + c + 16 * b);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float4 x = by[4 * b + e];
                            const float4 y = make_float4(fmaf(x.x, held, __uint_as_float(o[4 * e]) * fix), fmaf(x.y, held, __uint_as_float(o[4 * e + 1]) * fix),
                                                         fmaf(x.z, held, __uint_as_float(o[4 * e + 2]) * fix), fmaf(x.w, held, __uint_as_float(o[4 * e + 3]) * fix));
                            if (!end) sums[(c + 16 * b + 4 * e) * 8] = y;
                            o[4 * e] = __float_as_uint(y.x);
                            o[4 * e + 1] = __float_as_uint(y.y);
                            o[4 * e + 2] = __float_as_uint(y.z);
                            o[4 * e + 3] = __float_as_uint(y.w);
                        }
                        if (end) tmem_st16(ot + c + 16 * b, o);
                    }
                }
                if (end) tmem_wait_st();
                lw = cut = 0.f;
                held = 1.f;
            };
            // A tile's P from its S; FULL: no key of the tile is hidden from a row of the warp. The maximum is not
            // taken: p at most 2^8 is all that P needs, and a sum of the row's p at most 2^8 says so. A row whose
            // sum is above (its m is behind), or without an m yet, moves it and the warp takes the tile again.
            // Shared memory is slow while products read it (a poll or a shuffle takes some 200 clocks), so what does
            // not need S is done before the wait, and the next S is looked for in mid-tile.
            float kf[NB], vr[NB], vmax = 0.f;
            bool ready = false;
            auto tile = [&](auto whole, int i) {
                constexpr bool FULL = decltype(whole)::value;
                const int seen = limit - (j0 + i) * KT;
                const uint32_t sb = st + (i & 1) * KT;
                constexpr int AT = TERMS == 1 ? NB : 1;  // blocks read at once, as registers allow
                uint32_t hi[NB][16], lo[NB][16];
                float add, terms = 0.f;
                for (;;) {
                    const float mu = mref == -INFINITY ? 0.f : mref;
                    const uint64_t mu2 = pair(-mu, -mu);
                    uint64_t sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
                    uint32_t r[AT][32];
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        if (b % AT == 0) {
#pragma unroll
                            for (int k = 0; k < AT; ++k) tmem_ld32(r[k], sb + 32 * (b + k));
                            tmem_wait_ld();
                        }
                        if (b == NB - 1 && !ready && i + 1 < n) ready = bar_test(&bar->s_full[m][(i + 1) & 1], (uint32_t)((i + 1) >> 1) & 1);
                        const uint64_t kf2 = pair(kf[b], kf[b]), vr2 = pair(vr[b], vr[b]);
                        const int c = seen - 32 * b;
                        const uint32_t(&x)[32] = r[b % AT];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float p0, p1, w0, w1;
                            unpair(fma2(pair(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), kf2, mu2), p0, p1);
                            p0 = ex2(p0);
                            p1 = ex2(p1);
                            if (!FULL) {
                                if (2 * e >= c) p0 = 0.f;
                                if (2 * e + 1 >= c) p1 = 0.f;
                            }
                            const uint64_t p = pair(p0, p1);
                            uint64_t& to = sum[TERMS == 2 ? b : e & 1];
                            to = add2(to, p);
                            unpair(mul2(p, vr2), w0, w1);
                            if (!FULL) {  // (a scale that is not finite may lie behind a row's keys)
                                if (2 * e >= c) w0 = 0.f;
                                if (2 * e + 1 >= c) w1 = 0.f;
                            }
                            const __half2 h = __floats2half2_rn(w0, w1);
                            hi[b][e] = h2_bits(h);
                            const float2 f = __half22float2(h);
                            const float d0 = w0 - f.x, d1 = w1 - f.y;
                            lo[b][e] = h2_bits(__floats2half2_rn(d0, d1));
                        }
                    }
                    float s0, s1, s2, s3;
                    unpair(sum[0], s0, s1);
                    unpair(sum[1], s2, s3);
                    add = (s0 + s1) + (s2 + s3);
                    if (TERMS == 2)  // (a block behind the row's keys adds 0, whatever its scale)
                        terms = (s0 + s1 != 0.f ? (s0 + s1) * vr[0] : 0.f) + (s2 + s3 != 0.f ? (s2 + s3) * vr[NB - 1] : 0.f);
                    const float before = mref;
                    if (!__any_sync(0xffffffffu, add > kMostP)) break;
                    move(i, kf, vmax);
                    // (a score that is infinite leaves m where it is: its row is not a number)
                    if (!__any_sync(0xffffffffu, mref != before)) break;
                }
                l += add;
                if (TERMS == 2) {
                    lw += terms;
                    cut += kCut * lw;
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {  // over the block's scores: hi in its first 16 columns, lo in the next
                    tmem_st16(sb + 32 * b, hi[b]);
                    tmem_st16(sb + 32 * b + 16, lo[b]);
                }
            };
            for (int i = 0; i < n && alive; ++i) {
                const int seen = limit - (j0 + i) * KT;
                float vb[NB];
                vmax = 0.f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    kf[b] = factor * nk[b];
                    vb[b] = nv[b];
                    if (seen > 32 * b) vmax = fmaxf(vmax, vb[b]);
                }
                if (i + 1 < n) scales(j0 + i + 1);
                const bool moves = __any_sync(0xffffffffu, (mref == -INFINITY && seen > 0) || vmax > 4.f * vref);
                if (!__all_sync(0xffffffffu, ready)) {
                    alive = __all_sync(0xffffffffu, wait_or(&bar->s_full[m][i & 1], (uint32_t)(i >> 1) & 1, &bar->dead, a.err));
                    if (!alive) break;
                }
                ready = false;
                tc_after();
                if (moves || (i && i % kChain == 0)) {
                    if (i && i % kChain == 0) put_by(i, false);
                    if (moves) move(i, kf, vmax);
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) vr[b] = vb[b] == 0.f ? 0.f : __fdividef(vb[b], vref) * kPScale;
                if ((j0 + i + 1) * KT <= all) tile(std::true_type{}, i);
                else tile(std::false_type{}, i);
                tmem_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&bar->p_full[m][i & 1]);
            }
            // ---- the row's output, or its part ----
            if (n && alive) alive = __all_sync(0xffffffffu, wait_or(&bar->o_full[m], 0, &bar->dead, a.err));
            tc_after();
            if (n > kChain) put_by(n, true);
            const bool whole = sh.whole(), out = on;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const float up = (whole ? inv : 1.f) * vref * (1.f / kPScale) * (TERMS == 2 && lw != 0.f ? 1.f + cut / lw : 1.f);
            const size_t pr = ((size_t)kvh * rows + rr) * a.nsplit + split;
            const long long ob = (long long)(rr / a.group) * a.os + (long long)(kvh * a.group + rr % a.group) * hd;
            float* po = a.part_o + pr * hd;
#pragma unroll 2
            for (int c = 0; c < hd; c += 16) {
                uint32_t r[16];
                if (n) {
                    tmem_ld16(r, ot + c);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) r[e] = 0;
                }
                if (!out) continue;
                // a row that has seen no key, or only blocks of zeros: 0
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = l == 0.f ? 0.f : __uint_as_float(r[e]) * up;
                if (!whole) {
                    store16(po + c, v);
                } else {
                    T* d = (T*)a.o + ob + c;
                    alignas(16) T w[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) w[e] = from_f<T>(v[e]);
                    store16(d, w);
                }
            }
            if (out) {
                const float mu = mref == -INFINITY ? 0.f : mref;
                float* d = whole ? a.stats + ((size_t)kvh * rows + rr) * 2 : a.part_ml + pr * 2;
                d[0] = whole ? mu : mref;
                d[1] = whole ? inv : l;
            }
            tc_before();
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));  // whole warpgroups
        if (warp < kMmaWarp) {
            // ---- conversion: codes to fp16, swizzled ----
            constexpr int kConv = kConvWarps * 32;
            const int ct = tid - kSoftWarps * 32;
            const int pieces = hd / 16;                 // 16-byte pieces of a row
            const int total = KT * pieces;
            constexpr int L = (KT * PANELS * 4 + kConv - 1) / kConv;  // pieces per thread at most
            const uint4* kc = reinterpret_cast<const uint4*>(a.c.k + (size_t)kvh * cap * hd);
            const uint4* vc = reinterpret_cast<const uint4*>(a.c.v + (size_t)kvh * cap * hd);
            const long long end = (long long)cap * pieces;
            uint4 kr[L], vr[L];
            int put[L];  // where a piece goes in a tile
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const int p = ct + kConv * i, r = p / pieces;
                put[i] = p < total ? put_at(KT, r, p - r * pieces) : -1;
            }
            auto load = [&](uint4 (&w)[L], const uint4* base, int j) {
                const long long at = (long long)j * total + ct;
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    w[i] = make_uint4(0, 0, 0, 0);
                    if (put[i] >= 0 && at + kConv * i < end) w[i] = base[at + kConv * i];
                }
            };
            auto store = [&](const uint4 (&w)[L], unsigned char* d) {
#pragma unroll
                for (int i = 0; i < L; ++i)
                    if (put[i] >= 0) put_codes(d, put[i], w[i]);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            };
            if (most) {
                load(kr, kc, j0);
                load(vr, vc, j0);
            }
            for (int i = 0; i < most; ++i) {
                const int s = i % ST;
                const uint32_t ph = (uint32_t)(i / ST) & 1;
                if (i >= ST && !__all_sync(0xffffffffu, wait_or(&bar->k_empty[s], ph ^ 1, &bar->dead, a.err))) break;
                store(kr, ks + s * S::Stage);
                if (lane == 0) bar_arrive(&bar->k_full[s]);
                if (i + 1 < most) load(kr, kc, j0 + i + 1);
                if (i >= ST && !__all_sync(0xffffffffu, wait_or(&bar->v_empty[s], ph ^ 1, &bar->dead, a.err))) break;
                store(vr, vs + s * S::Stage);
                if (lane == 0) bar_arrive(&bar->v_full[s]);
                if (i + 1 < most) load(vr, vc, j0 + i + 1);
            }
        } else if (warp - kMmaWarp < MT && (most || (a.weight && split == 0))) {
            // ---- products: a warp per query tile (a poll takes some 200 clocks while products read shared
            // memory; the other tile's products run meanwhile). The whole warp goes along and one elected lane
            // issues; descriptors come from one shuffled word each, so they stay in uniform registers ----
            const uint32_t id_s = instr(KT, false), id_o = instr(hd, true);
            const int steps = hd / 16, m = uniform(warp - kMmaWarp);
            const uint32_t base = uniform(smem_addr(qs)), qb = base + m * S::QTile;
            const uint32_t kb = base + MT * S::QTile, vb = kb + ST * S::Stage;
            const int n = uniform(m == 0 ? nt[0] : nt[MT - 1]), all = uniform(most);
            const uint32_t tm = uniform(tmem), ts = tm + m * S::SCols, to = tm + MT * S::SCols + m * S::OCols;
            auto wait = [&](uint64_t* b, uint32_t parity) {
                bool ok = true;
                if (lane == 0) ok = wait_or(b, parity, &bar->dead, a.err);
                return uniform((int)ok) != 0;
            };
            auto wait_k = [&](int t) { return wait(&bar->k_full[t % ST], (uint32_t)(t / ST) & 1); };
            auto scores = [&](int t) {  // S = Q K^T of the share's tile t
                const uint32_t k = uniform(operand_lo(kb + t % ST * S::Stage, 16)), q = uniform(operand_lo(qb, 16));
                const uint32_t d = uniform(ts + (t & 1) * KT);
                if (elected()) {
                    // the lo terms first: each product's sum is cut off, which then costs them nothing
                    auto step = [&](int x, int s) {
                        mma_ss(d, operand_of(q + ((TERMS - 1 - x) * PANELS + (s >> 2)) * 1024 + (s & 3) * 2),
                               operand_of(k + (s >> 2) * (KT * 8) + (s & 3) * 2), id_s, x + s > 0);
                    };
                    if (steps == PANELS * 4) {
#pragma unroll
                        for (int x = 0; x < TERMS; ++x)
#pragma unroll
                            for (int s = 0; s < PANELS * 4; ++s) step(x, s);
                    } else {
#pragma unroll 1
                        for (int x = 0; x < TERMS; ++x)
#pragma unroll 1
                            for (int s = 0; s < steps; ++s) step(x, s);
                    }
                    tc_commit(&bar->s_full[m][t & 1]);
                    tc_commit(&bar->k_empty[t % ST]);
                }
            };
            auto output = [&](int t) {  // O (+)= P V; P of key block b: hi at columns 32 b, lo 16 on
                const uint32_t v = uniform(operand_lo(vb + t % ST * S::Stage, KT * 128));
                const uint32_t p = uniform(ts + (t & 1) * KT);
                if (elected()) {
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int s = 0; s < KT / 16; ++s)
                            mma_ts(to, p + 32 * (s >> 1) + 16 * x + 8 * (s & 1), operand_of(v + s * 128), id_o, t % kChain || x + s > 0);
                    tc_commit(&bar->o_done[m]);
                    tc_commit(&bar->v_empty[t % ST]);
                    if (t + 1 == n) tc_commit(&bar->o_full[m]);
                }
            };
            bool alive = wait(&bar->q, 0);
            const bool keep = a.weight && split == 0 && alive;
            if (keep && lane == 0) {  // the weights' kernel reads the query tiles
                unsigned char* dst = a.qt + ((size_t)kvh * tiles128 + (size_t)unit * MT + m) * S::QTile;
                for (int p = 0; p < TERMS * PANELS; ++p)
                    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst + (size_t)p * 16384),
                                 "r"(qb + p * 16384), "r"(16384)
                                 : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
#pragma unroll 1
            for (int t = 0; t < S::Ahead && t < n && alive; ++t) {
                alive = wait_k(t);
                tc_after();
                if (alive) scores(t);
            }
#pragma unroll 1
            for (int i = 0; alive && i < n; ++i) {
                // K of a later tile has come after V of this one
                const int t = i + S::Ahead;
                alive = (t < n ? wait_k(t) : wait(&bar->v_full[i % ST], (uint32_t)(i / ST) & 1)) &&
                        wait(&bar->p_full[m][i & 1], (uint32_t)(i >> 1) & 1);
                if (!alive) break;
                tc_after();
                output(i);
                if (t < n) scores(t);
            }
            // tiles that this query tile does not need: passed on
            if (alive && lane == 0)
                for (int t = n; t < all; ++t) {
                    alive = wait_or(&bar->v_full[t % ST], (uint32_t)(t / ST) & 1, &bar->dead, a.err);
                    if (!alive) break;
                    bar_arrive(&bar->k_empty[t % ST]);
                    bar_arrive(&bar->v_empty[t % ST]);
                }
            // every product has ended before tensor memory is freed
            if (elected()) tc_commit(&bar->drain[m]);
            volatile int never = 0;
            if (lane == 0) wait_or(&bar->drain[m], 0, &never, a.err);
            if (keep && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    }
    __syncwarp();
    tc_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_after();
        tmem_free(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// The cached rows' weights: a CTA keeps MT tiles of 128 keys (their codes as
// fp16) and streams the query tiles, S = Q K^T. A thread has one query of each
// tile and 32 MT keys; it adds p = 2^(t - m) / l = 2^(s factor scale - (m + log2 l))
// to its keys' sums in registers, over all tiles, and the 128 queries of a key
// are added up once, at the end, in a fixed order. The keys are two halves with
// two buffers of S each, and the second half follows a tile behind, so the
// warps of one take the exponentials while those of the other wait. Needs the
// rows' final m, 1 / l.
// exp2 bounds it, one per key and query: 4008 rows over 30501 keys of four heads
// take 232 us where the exponentials alone are 115 us (16 a clock and SM); the
// last of four waves of CTAs is a quarter full, and a tile takes 3300 cycles of
// which 2050 are exponentials. A thread with one key and all queries (S^T)
// reads each query's numbers from shared memory: 255 us, and 247 us with twice
// the warps; both halves of the keys in step 240 us.
// ---------------------------------------------------------------------------
template <int PANELS>
struct WShape {
    static constexpr int MT = PANELS <= 2 ? 2 : 1;
    static constexpr int Keys = MT * 128;
    static constexpr int KTile = PANELS * Keys * 128;  // the keys
    static constexpr int Stage = PANELS * 16384;       // a query tile's hi or lo terms
    static constexpr int ST = PANELS <= 2 ? 4 : 2;
    static constexpr int Smem = KTile + ST * Stage + 4 * Keys * 4 + 1024 + 256;
    static_assert(Smem <= 232448, "shared memory");
};
// warps 0-15 convert the keys, then sum: four of them share a quarter of the keys; 16 the products, 17 loads
constexpr int kWSumWarps = 16, kWMmaWarp = 16, kWThreads = 576;

struct WBars {
    uint64_t k_full, q_full[4], q_empty[4], s_full[2][2], s_empty[2][2], drain;
    uint32_t tmem;
    int dead;
};
static_assert(sizeof(WBars) <= 256, "barriers");

template <int PANELS, int TERMS>
__global__ void __launch_bounds__(kWThreads, 1) kv8_prompt_weight_kernel(const __grid_constant__ AttnArgs a, int tiles128) {
    using S = WShape<PANELS>;
    constexpr int ST = S::ST, Keys = S::Keys, KC = Keys / 4;
    constexpr int Lag = 2 * TERMS <= ST ? 1 : 0;  // (the ring holds two query tiles)
    extern __shared__ unsigned char raw[];
    pdl_wait();
    pdl_trigger();
    const int hd = (int)a.c.head_dim, cap = (int)a.c.capacity, rows = a.n * a.group, kvh = blockIdx.y;
    const int past = *a.c.past, keys = keys_of(past, a.n - 1, cap);
    const int key0 = blockIdx.x * Keys;
    if (key0 >= keys) return;
    unsigned char* smem = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    unsigned char *ks = smem, *qs = ks + S::KTile;
    float* part = reinterpret_cast<float*>(qs + ST * S::Stage);  // [4][Keys]
    WBars* bar = reinterpret_cast<WBars*>(part + 4 * Keys);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (warp == kWMmaWarp) {
        if (lane == 0) {
            bar_init(&bar->k_full, kWSumWarps);
            for (int i = 0; i < ST; ++i) {
                bar_init(&bar->q_full[i], 1);
                bar_init(&bar->q_empty[i], 1);
            }
            for (int i = 0; i < 4; ++i) {
                bar_init(&bar->s_full[i >> 1][i & 1], 1);
                bar_init(&bar->s_empty[i >> 1][i & 1], kWSumWarps / 2);
            }
            bar_init(&bar->drain, 1);
            bar->dead = 0;
            bar_init_fence();
        }
        __syncwarp();
        tmem_alloc(&bar->tmem, 2 * Keys);
        tc_before();
    }
    __syncthreads();
    tc_after();
    const uint32_t tmem = bar->tmem;
    // query tiles from the first row that sees key0
    const int first = (int)min((long long)rows - 1, max(0LL, ((long long)key0 - past) * a.group)) / 128;
    const int n = (rows + 127) / 128 - first;

    if (warp < kWSumWarps) {
        const int pieces = hd / 16;
        const uint4* kc = reinterpret_cast<const uint4*>(a.c.k + ((size_t)kvh * cap + key0) * hd);
        const int held = min(Keys, cap - key0) * pieces;
        for (int p = tid; p < Keys * pieces; p += kWSumWarps * 32) {
            const int r = p / pieces;
            const uint4 w = p < held ? kc[p] : make_uint4(0, 0, 0, 0);
            put_codes(ks, put_at(Keys, r, p - r * pieces), w);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(&bar->k_full);

        const int quarter = warp & 3, half = warp >> 3, cols = (warp >> 2) * KC, base = key0 + cols;
        const uint32_t st = tmem + ((uint32_t)quarter << 21) + cols;
        float scale[KC / 32];
#pragma unroll
        for (int h = 0; h < KC / 32; ++h) scale[h] = base + 32 * h < keys ? a.c.k_scale[(size_t)kvh * (cap >> 5) + (base >> 5) + h] : 0.f;
        uint64_t sum[KC / 2];
#pragma unroll
        for (int e = 0; e < KC / 2; ++e) sum[e] = pair(0.f, 0.f);
        // a row's factor, m and 1 / l (0 for a row without keys: p = 0); the next tile's are on their way while a
        // tile is summed
        float factor;
        float2 ml;
        auto numbers = [&](int i) {
            const int r = (first + i) * 128 + quarter * 32 + lane;
            factor = 0.f;
            ml = make_float2(0.f, 0.f);
            if (i < n && r < rows) {
                ml = *reinterpret_cast<const float2*>(a.stats + ((size_t)kvh * rows + r) * 2);
                factor = a.qfactor[(size_t)kvh * tiles128 * 128 + r];
            }
        };
        numbers(0);
        for (int i = 0; i < n; ++i) {
            const int b = i & 1, r0 = (first + i) * 128 + quarter * 32;
            const float mine = factor, less = log2f(ml.y) - ml.x;  // -(m + log2 l)
            numbers(i + 1);
            const bool ok = wait_or(&bar->s_full[half][b], (uint32_t)((i >> 1) & 1), &bar->dead, a.err);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_after();
            const bool full = (long long)past + r0 / a.group >= base + KC - 1;
            const long long left = (long long)past + (r0 + lane) / a.group - base;  // the last column that this row sees
            const uint64_t minus = pair(less, less);
#pragma unroll
            for (int h = 0; h < KC / 16; ++h) {
                uint32_t r[16];
                tmem_ld16(r, st + b * Keys + 16 * h);
                const float f = mine * scale[h / 2];
                const uint64_t ff = pair(f, f);
                tmem_wait_ld();
                if (full) {
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        float p0, p1;
                        unpair(fma2(pair(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), ff, minus), p0, p1);
                        sum[8 * h + e / 2] = add2(sum[8 * h + e / 2], pair(ex2(p0), ex2(p1)));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        float p0, p1;
                        unpair(fma2(pair(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), ff, minus), p0, p1);
                        p0 = 16 * h + e <= left ? ex2(p0) : 0.f;
                        p1 = 16 * h + e + 1 <= left ? ex2(p1) : 0.f;
                        sum[8 * h + e / 2] = add2(sum[8 * h + e / 2], pair(p0, p1));
                    }
                }
            }
            tc_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&bar->s_empty[half][b]);
        }
        // the warp's 32 rows: each step adds the lanes that differ in one bit and halves what a lane has
        float v[KC];
#pragma unroll
        for (int e = 0; e < KC / 2; ++e) unpair(sum[e], v[2 * e], v[2 * e + 1]);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) {
            const int c = KC * w / 32;
            const bool up = lane & w;
#pragma unroll
            for (int e = 0; e < c; ++e) {
                const float keep = up ? v[e + c] : v[e], give = up ? v[e] : v[e + c];
                v[e] = keep + __shfl_xor_sync(0xffffffffu, give, w);
            }
        }
#pragma unroll
        for (int e = 0; e < KC / 32; ++e) part[quarter * Keys + cols + lane * (KC / 32) + e] = v[e];
    } else if (warp == kWMmaWarp) {
        const uint32_t id = instr(Keys / 2, false), tm = uniform(tmem), base = uniform(smem_addr(ks));
        const int steps = hd / 16, count = uniform(n);
        auto wait = [&](uint64_t* w, uint32_t parity) {
            bool ok = true;
            if (lane == 0) ok = wait_or(w, parity, &bar->dead, a.err);
            return uniform((int)ok) != 0;
        };
        bool ok = wait(&bar->k_full, 0);
        for (int j = 0; ok && j < 2 * (count + Lag); ++j) {
            const int half = j & 1, i = (j >> 1) - half * Lag, b = i & 1;
            if (i < 0 || i >= count) continue;
            if (i >= 2) ok = wait(&bar->s_empty[half][b], (uint32_t)((i >> 1) & 1) ^ 1);
            for (int t = 0; ok && t < TERMS; ++t) {
                const int it = i * TERMS + t, sg = it % ST;
                ok = wait(&bar->q_full[sg], (uint32_t)((it / ST) & 1));
                if (!ok) break;
                tc_after();
                // (a row is 8 of the operand's units: to the half's first row)
                const uint32_t k = uniform(operand_lo(base, 16) + half * (Keys / 2 * 8));
                const uint32_t q = uniform(operand_lo(base + S::KTile + sg * S::Stage, 16));
                const uint32_t d = uniform(tm + b * Keys + half * (Keys / 2));
                const bool add = t > 0;
                if (elected()) {
#pragma unroll
                    for (int s = 0; s < PANELS * 4; ++s)
                        if (s < steps)
                            mma_ss(d, operand_of(q + (s >> 2) * 1024 + (s & 3) * 2), operand_of(k + (s >> 2) * (Keys * 8) + (s & 3) * 2), id,
                                   add || s > 0);
                    if (half) tc_commit(&bar->q_empty[sg]);
                }
            }
            if (ok && elected()) tc_commit(&bar->s_full[half][b]);
        }
        if (elected()) tc_commit(&bar->drain);
        volatile int never = 0;
        if (lane == 0) wait_or(&bar->drain, 0, &never, a.err);
    } else if (lane == 0) {
        const unsigned char* src = a.qt + ((size_t)kvh * tiles128 + first) * TERMS * S::Stage;  // (a tile's lo terms first)
        const int total = n * TERMS;
        int it = 0;
        for (; it < total; ++it) {
            const int sg = it % ST;
            if (it >= ST && !wait_or(&bar->q_empty[sg], (uint32_t)((it / ST) & 1) ^ 1, &bar->dead, a.err)) break;
            bar_expect(&bar->q_full[sg], S::Stage);
            bulk_load(qs + sg * S::Stage, src + (size_t)(it / TERMS * TERMS + TERMS - 1 - it % TERMS) * S::Stage, S::Stage, &bar->q_full[sg]);
        }
        // the copies in flight end before this CTA's shared memory does
        volatile int never = 0;
        for (int k = max(0, it - ST); k < it; ++k) wait_or(&bar->q_full[k % ST], (uint32_t)((k / ST) & 1), &never, a.err);
    }
    __syncwarp();
    tc_before();
    __syncthreads();
    if (tid < Keys && key0 + tid < keys) {
        const float v = (part[tid] + part[Keys + tid]) + (part[2 * Keys + tid] + part[3 * Keys + tid]);
        float* w = a.weight + (size_t)kvh * cap + key0 + tid;
        *w = key0 + tid < past ? *w + v : v;
    }
    if (warp == kWMmaWarp) {
        tc_after();
        tmem_free(tmem, 2 * Keys);
    }
}

template <int PANELS, int TERMS>
int launch_weights(const AttnArgs& a, cudaStream_t st) {
    using S = WShape<PANELS>;
    auto k = kv8_prompt_weight_kernel<PANELS, TERMS>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::Smem);
    if (e != cudaSuccess) return neon_internal::cuda_error(e, "cudaFuncSetAttribute(kv8_prompt_weight_kernel)");
    const int tiles = (a.n * a.group + 255) / 256 * 2;
    const unsigned grid = (a.c.capacity + S::Keys - 1) / S::Keys;
    return launch("kv8_prompt_weight_kernel", k, dim3(grid, a.c.n_kv_head), kWThreads, S::Smem, st, 1, a, tiles);
}

using PromptKernel = void (*)(AttnArgs, int);

template <int PANELS, typename T>
int launch_shape(const AttnArgs& a, cudaStream_t st) {
    using S = Shape<PANELS, sizeof(T) == 4 ? 2 : 1>;
    const int rows = a.n * a.group, H = (int)a.c.n_kv_head;
    const int tiles = (rows + 255) / 256 * 2;
    PromptKernel k = kv8_prompt_kernel<PANELS, T>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::Smem);
    if (e != cudaSuccess) return neon_internal::cuda_error(e, "cudaFuncSetAttribute(kv8_prompt_kernel)");
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, k);
    if (e != cudaSuccess) return neon_internal::cuda_error(e, "cudaFuncGetAttributes(kv8_prompt_kernel)");
    // the register split would wait for registers that the launch did not bring
    if (fa.numRegs < kLaunchRegs) return neon_internal::error(NEON_ERR_UNSUPPORTED, "kv8_prompt_kernel: built with too few registers");
    const int units = (rows + 128 * S::MT - 1) / (128 * S::MT);
    return launch("kv8_prompt_kernel", k, dim3((unsigned)(units * H * a.nsplit)), kThreads, S::Smem, st, 1, a, tiles);
}

}  // namespace

int prompt_unit(int hd) { return hd <= 128 ? 256 : 128; }
int prompt_tile_shift() { return kTileShift; }

size_t prompt_query_bytes(const neon_kv8_t& c, size_t rows, int type) {
    const size_t tiles = (rows + 255) / 256 * 2, panels = (c.head_dim + 63) / 64;
    return c.n_kv_head * tiles * (type == NEON_GGML_F32 ? 2 : 1) * panels * 16384;
}

template <int PANELS>
static int launch_typed(const AttnArgs& a, cudaStream_t st) {
    return a.type == NEON_GGML_F32   ? launch_shape<PANELS, float>(a, st)
           : a.type == NEON_GGML_F16 ? launch_shape<PANELS, __half>(a, st)
                                     : launch_shape<PANELS, __nv_bfloat16>(a, st);
}

int launch_prompt(const AttnArgs& a, cudaStream_t st) {
    switch (((int)a.c.head_dim + 63) / 64) {
        case 1: return launch_typed<1>(a, st);
        case 2: return launch_typed<2>(a, st);
        case 3: return launch_typed<3>(a, st);
        default: return launch_typed<4>(a, st);
    }
}

int launch_prompt_weights(const AttnArgs& a, cudaStream_t st) {
    const int panels = ((int)a.c.head_dim + 63) / 64;
    const bool two = a.type == NEON_GGML_F32;
    switch (panels) {
        case 1: return two ? launch_weights<1, 2>(a, st) : launch_weights<1, 1>(a, st);
        case 2: return two ? launch_weights<2, 2>(a, st) : launch_weights<2, 1>(a, st);
        case 3: return two ? launch_weights<3, 2>(a, st) : launch_weights<3, 1>(a, st);
        default: return two ? launch_weights<4, 2>(a, st) : launch_weights<4, 1>(a, st);
    }
}

}  // namespace longctx

