// neon_kv8_attn.cu -- attention over the KV cache in 8 bits
// (neon_cuda_kv8_attention).
//
//   t_ij = log2(e) scale s_k(block of j) (q_i . c_j),  p_ij = 2^(t_ij - m_i)
//   o_i = sum_j p_ij s_v(block of j) c'_j / sum_j p_ij,  weight_j += sum_i p_ij / l_i
//
// The codes are exact in 16-bit floats, so both products run on the tensor
// cores with fp32 sums, and only the other operand is rounded: fp32 values are
// split into two fp16 terms (hi + lo, 22 bits), of which every product is
// exact. Scales are applied in fp32 to the scores, and to p before the second
// product, where p is scaled so that its split keeps its bits (see kPUp).
#include "neon_kv8_attn.cuh"

#include <algorithm>

namespace longctx {
namespace {

// p (at most 2^8, times s_v over a reference that it is at most four times of)
// is multiplied by 2^5 before its split: hi stays below fp16's 65504, and lo
// keeps values down to 2^-30 of the row's largest.
constexpr float kPUp = 32.f, kPDown = 1.f / 32.f;

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr size_t kSms = 148;    // of a B200: a constant, as a workspace is sized without a device
constexpr int kMaxSplit = 64;  // (one KV head over 60000 rows takes 25.6 us; with 32 shares 27.8)

// ---------------------------------------------------------------------------
// Eight or sixteen rows of one KV head over a share of the cache. The MMA's 16
// rows hold eight rows' hi terms and below them their lo terms, so the split
// costs no extra products: a row's score is the sum of its two halves, and its
// output likewise. Of more than eight rows in a 16-bit type they hold sixteen
// rows' single terms (q is exact in one, up to values far below the row's
// largest), and p's lo terms take a second product: 16 rows over 120000 of 8
// heads x 128 take 69 us where two passes of eight took 95, and 32 rows 112
// where four took 186 (with p rounded to one term, 2^-11 of itself: 63 and 100).
// Each warp streams its own tiles of 32 rows (a block of the
// cache: K's codes, then V's, a bulk copy each) through its own ring in shared
// memory, with no barrier between the warps until their results are merged.
// The order of the summed dimension is free, so each lane reads whole 16-byte
// pieces of a K row and the query fragments (in shared memory, the same for
// all warps) are laid out to match; of V, lane group g takes columns [g HD / 8,
// (g + 1) HD / 8) of four rows. HBM bounds it at length; the arithmetic (some
// 800 instructions a warp for 8 KB of codes) needs 16 warps per SM to hide its
// latencies: 131071 rows of 8 heads x 128 take 66 us with the weights' scores
// stored, of which the stream is 47 (5.8 TB/s) and the rest prologue, merge and
// the last warps; with 8 warps, and the query fragments in registers, 68 us
// without.
// ---------------------------------------------------------------------------
template <int HD, int ROWS>
struct RowTile {
    static constexpr int kWarps = HD <= 128 ? 16 : 8;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kSlots = HD <= 64 ? 6 : 3;
    static constexpr int kSlotBytes = 32 * HD;
    static constexpr int kRing = kWarps * kSlots * kSlotBytes;
    static constexpr int kPitch = HD + 8;  // floats of a row in the merge: eight rows in different banks
    static constexpr int kMerge = kWarps * ROWS * (kPitch + 2) * 4;
    static constexpr int kBody = kRing > kMerge ? kRing : kMerge;
    static constexpr int kQuery = HD / 16 * 512;
    static constexpr int kSmem = kBody + kQuery + 16 * 4 + kWarps * kSlots * 8;
    static_assert(kSmem <= 232448, "shared memory");
};

// The query fragments of row g of a group, by a warp: lane (g % 8, tq) of the products holds values
// tq HD / 4 + 4 s .. + 3 of row g for step s, as hi and lo terms (of 16 rows: row g's and row g + 8's values), times
// 2^e so that the row's largest is near 2^7 (its lo terms then stay normal halves, and of a 16-bit type only values
// below 2^-20 of the row's largest lose bits). The row's factor is scale log2(e) 2^-e.
template <int HD, int ROWS>
__device__ __forceinline__ void row_queries(const AttnArgs& a, int kvh, int grp, int g, uint4* out, float* factor) {
    const int lane = threadIdx.x & 31, hd = (int)a.c.head_dim, rows = a.n * a.group, row = grp * ROWS + g;
    const int tok = token_of(a, row);
    const long long base = tok * a.qs + (long long)(kvh * a.group + row - tok * a.group) * hd;
    constexpr int V = (HD + 127) / 128;  // pieces of four values a lane
    float x[V][4];
    float mx = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 4 * (lane + 32 * v) + i;
            x[v][i] = row < rows && d < hd ? q_value(a.q, a.type, base + d) : 0.f;
        }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fabsf(x[v][i]));
    const unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(mx)) >> 23;
    const int e = top >= 255u ? 0 : min(120, 134 - (int)top);
    const float f = pow2(e);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int d = 4 * (lane + 32 * v);
        if (d >= HD) continue;
        uint4 q;
        split2(x[v][0] * f, x[v][1] * f, q.x, q.y);
        split2(x[v][2] * f, x[v][3] * f, q.z, q.w);
        uint4* to = out + d % (HD / 4) / 4 * 32 + g % 8 * 4 + d / (HD / 4);
        if (ROWS == 8) {
            *to = q;
        } else {
            uint32_t* half = reinterpret_cast<uint32_t*>(to) + g / 8;
            half[0] = q.x;
            half[2] = q.z;
        }
    }
    if (lane == 0) factor[g] = a.scale * pow2(-e);
}

// FULL: head_dim is HD itself, not less.
template <int HD, bool FULL, int ROWS>
__global__ void __launch_bounds__(RowTile<HD, ROWS>::kThreads, 1) kv8_rows_kernel(const __grid_constant__ AttnArgs a) {
    using R = RowTile<HD, ROWS>;
    constexpr int RL = ROWS / 8;  // rows of a lane: g, and of 16 g + 8
    constexpr int NT = HD / 8;    // column tiles of the output
    constexpr int W = R::kWarps, S = R::kSlots;
    extern __shared__ __align__(128) unsigned char smem[];
    uint4* qf = reinterpret_cast<uint4*>(smem + R::kBody);
    float* qfac = reinterpret_cast<float*>(smem + R::kBody + R::kQuery);
    uint64_t* bars = reinterpret_cast<uint64_t*>(qfac + 16);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
    const int hd = FULL ? HD : (int)a.c.head_dim, cap = (int)a.c.capacity;
    const int split = blockIdx.x, kvh = blockIdx.y, grp = blockIdx.z, rows = a.n * a.group;
    unsigned char* ring = smem + warp * S * R::kSlotBytes;
    uint64_t* bar = bars + warp * S;
    if (lane == 0) {
        for (int s = 0; s < S; ++s) bar_init(&bar[s], 1);
        bar_init_fence();
    }
    __syncwarp();
    pdl_wait();
    pdl_trigger();

    // the keys of the group's rows, and this warp's share of them in tiles
    const int past = *a.c.past;
    int limit[RL];
#pragma unroll
    for (int h = 0; h < RL; ++h) {
        const int row = grp * ROWS + 8 * h + g;
        limit[h] = row < rows ? keys_of(past, token_of(a, row), cap) : 0;
    }
    const Shares sh = shares_of(a, past, grp);
    if (!sh.has(split)) return;
    const int c0 = split * sh.per, c1 = min(c0 + sh.per, sh.tiles);
    const int per_warp = (c1 - c0 + W - 1) / W;
    const int w0 = min(c0 + warp * per_warp, c1), w1 = min(w0 + per_warp, c1);

    const int8_t* kc = a.c.k + (size_t)kvh * cap * hd;
    const int8_t* vc = a.c.v + (size_t)kvh * cap * hd;
    const float* ksc = a.c.k_scale + (size_t)kvh * (cap >> 5);
    const float* vsc = a.c.v_scale + (size_t)kvh * (cap >> 5);
    const uint32_t bytes = 32u * hd;
    const int items = 2 * (w1 - w0);  // K of a tile, then its V
    auto issue = [&](int it, int slot) {
        bar_expect(&bar[slot], bytes);
        bulk_load(ring + slot * R::kSlotBytes, (it & 1 ? vc : kc) + (size_t)(w0 + (it >> 1)) * bytes, bytes, &bar[slot]);
    };
    if (lane == 0)
        for (int it = 0; it < min(S, items); ++it) issue(it, it);
    for (int r = warp; r < ROWS; r += W) row_queries<HD, ROWS>(a, kvh, grp, r, qf, qfac);
    __syncthreads();
    float factor[RL];
#pragma unroll
    for (int h = 0; h < RL; ++h) factor[h] = qfac[8 * h + g];
    float* scores = a.scores ? a.scores + (((size_t)kvh * gridDim.z + grp) * ROWS + g) * cap : nullptr;

    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    float m[RL], l[RL], vref = 0.f;
#pragma unroll
    for (int h = 0; h < RL; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
    }
    float my_ks = 0.f, my_vs = 0.f;  // the scales of 32 tiles, one per lane
    bool ok = true;
    int slot = 0;
    uint32_t phase = 0;
    auto take = [&]() {  // waits for the next item
        ok = __all_sync(0xffffffffu, bar_wait(&bar[slot], phase, a.err));
        return ring + slot * R::kSlotBytes;
    };
    auto give = [&](int it) {  // its slot goes to the item S further on
        __syncwarp();
        if (lane == 0 && it + S < items) issue(it + S, slot);
        if (++slot == S) {
            slot = 0;
            phase ^= 1;
        }
    };
    int it = 0;
    for (int tile = w0; tile < w1; ++tile) {
        const int at = (tile - w0) & 31;
        if (at == 0) {
            const int b = tile + lane;
            my_ks = b < w1 ? ksc[b] : 0.f;
            my_vs = b < w1 ? vsc[b] : 0.f;
        }
        const float ks = __shfl_sync(0xffffffffu, my_ks, at), vs = __shfl_sync(0xffffffffu, my_vs, at);
        const unsigned char* kt = take();
        if (!ok) break;

        // scores of 32 keys: key 8 j + g of column tile j
        float sc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[j][e] = 0.f;
#pragma unroll
        for (int p = 0; p < HD / 64; ++p) {
            uint4 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = make_uint4(0, 0, 0, 0);
                if (tq * (HD / 4) + 16 * p < hd)
                    w[j] = *reinterpret_cast<const uint4*>(kt + (8 * j + g) * hd + tq * (HD / 4) + 16 * p);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 qv = qf[(4 * p + i) * 32 + lane];
                const uint32_t q[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t u = (i == 0 ? w[j].x : i == 1 ? w[j].y : i == 2 ? w[j].z : w[j].w) ^ 0x80808080u;
                    mma16816(sc[j], q, codes_lo(u), codes_hi(u));
                }
            }
        }
        give(it++);
        // online softmax of the lane's rows: it has keys 8 j + 2 tq and + 1
        float t[RL][4][2], mu[RL], down[RL];
        bool moves = vs > 4.f * vref;
#pragma unroll
        for (int h = 0; h < RL; ++h) {
            const float kf = factor[h] * ks;
            float mt = m[h];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = tile * 32 + 8 * j + 2 * tq + e;
                    t[h][j][e] = key < limit[h] ? (ROWS == 8 ? sc[j][e] + sc[j][e + 2] : sc[j][e + 2 * h]) * kf : -INFINITY;
                    mt = fmaxf(mt, t[h][j][e]);
                }
            if (scores && grp * ROWS + 8 * h + g < rows)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *reinterpret_cast<float2*>(scores + (size_t)(8 * h) * cap + tile * 32 + 8 * j + 2 * tq) =
                        make_float2(t[h][j][0], t[h][j][1]);
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
            // m follows when p would pass 2^8 (the result does not depend on m): O is seldom rescaled
            const float mnew = mt > m[h] + 8.f || m[h] == -INFINITY ? mt : m[h];
            mu[h] = mnew == -INFINITY ? 0.f : mnew;
            down[h] = ex2(m[h] - mu[h]);
            moves |= mnew != m[h];
            m[h] = mnew;
        }
        if (__any_sync(0xffffffffu, moves)) {
            const float vtop = vs > 4.f * vref ? vs : vref;
            const float vdown = vtop > 0.f ? vref / vtop : 1.f;
            vref = vtop;
            float f[RL];
#pragma unroll
            for (int h = 0; h < RL; ++h) {
                l[h] *= down[h];
                f[h] = down[h] * vdown;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][e] *= f[ROWS == 8 ? 0 : e >> 1];
        }
        const float vr = vs == 0.f ? 0.f : vs / vref * kPUp;
        uint32_t pf[2][4], pl[2][ROWS == 16 ? 4 : 1];  // p's terms: of eight rows both in pf, of sixteen hi and lo
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int j = 2 * k + hf;
#pragma unroll
                for (int h = 0; h < RL; ++h) {
                    const bool on0 = t[h][j][0] != -INFINITY, on1 = t[h][j][1] != -INFINITY;
                    const float p0 = ex2(t[h][j][0] - mu[h]), p1 = ex2(t[h][j][1] - mu[h]);
                    l[h] += p0 + p1;
                    const float x0 = on0 ? p0 * vr : 0.f, x1 = on1 ? p1 * vr : 0.f;
                    if constexpr (ROWS == 8) split2(x0, x1, pf[k][2 * hf], pf[k][2 * hf + 1]);
                    else split2(x0, x1, pf[k][2 * hf + h], pl[k][2 * hf + h]);
                }
            }
        }
        const unsigned char* vt = take();
        if (!ok) break;
        // o += p V: lane (g, tq) reads columns g HD / 8 .. of rows 16 k + 2 tq, + 1, + 8, + 9
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const unsigned char* vrow = vt + (16 * k + 2 * tq) * hd + g * (HD / 8);
            constexpr int WD = HD / 32;  // words of a lane's columns
            uint32_t w[4][WD];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned char* src = vrow + ((r & 1) + 8 * (r >> 1)) * hd;
                if constexpr (WD == 2) {
                    uint2 v = make_uint2(0, 0);
                    if (g * 8 < hd) v = *reinterpret_cast<const uint2*>(src);
                    w[r][0] = v.x ^ 0x80808080u;
                    w[r][1] = v.y ^ 0x80808080u;
                } else {
#pragma unroll
                    for (int p = 0; p < WD / 4; ++p) {
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (g * (HD / 8) + 16 * p < hd) v = *reinterpret_cast<const uint4*>(src + 16 * p);
                        w[r][4 * p] = v.x ^ 0x80808080u;
                        w[r][4 * p + 1] = v.y ^ 0x80808080u;
                        w[r][4 * p + 2] = v.z ^ 0x80808080u;
                        w[r][4 * p + 3] = v.w ^ 0x80808080u;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < WD; ++i) {
                // bytes (r0 c0, r1 c0, r0 c1, r1 c1) and (.. c2, .. c3) of both row pairs
                const uint32_t a01 = __byte_perm(w[0][i], w[1][i], 0x5140), a23 = __byte_perm(w[0][i], w[1][i], 0x7362);
                const uint32_t b01 = __byte_perm(w[2][i], w[3][i], 0x5140), b23 = __byte_perm(w[2][i], w[3][i], 0x7362);
                mma16816(acc[4 * i], pf[k], codes_lo(a01), codes_lo(b01));
                mma16816(acc[4 * i + 1], pf[k], codes_hi(a01), codes_hi(b01));
                mma16816(acc[4 * i + 2], pf[k], codes_lo(a23), codes_lo(b23));
                mma16816(acc[4 * i + 3], pf[k], codes_hi(a23), codes_hi(b23));
                if constexpr (ROWS == 16) {
                    mma16816(acc[4 * i], pl[k], codes_lo(a01), codes_lo(b01));
                    mma16816(acc[4 * i + 1], pl[k], codes_hi(a01), codes_hi(b01));
                    mma16816(acc[4 * i + 2], pl[k], codes_lo(a23), codes_lo(b23));
                    mma16816(acc[4 * i + 3], pl[k], codes_hi(a23), codes_hi(b23));
                }
            }
        }
        give(it++);
    }
    if (!ok)  // this warp's copies in flight end (each wait bounded) before shared memory is reused
        for (int s = 0; s < min(S - 1, items - it - 1); ++s) {
            if (++slot == S) {
                slot = 0;
                phase ^= 1;
            }
            bar_wait(&bar[slot], phase, a.err);
        }

    // merge the warps: o (times s_v), m, l of each row
    __syncthreads();
    float* mo = reinterpret_cast<float*>(smem);             // [warps][ROWS][HD]: place 8 t + c has column c HD / 8 + t
    float* ml = mo + W * ROWS * R::kPitch;                  // [warps][ROWS][2]
    const float up = vref * kPDown;
#pragma unroll
    for (int h = 0; h < RL; ++h) {
        const int at = warp * ROWS + 8 * h + g;
        float* mine = mo + at * R::kPitch + 2 * tq;
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
#pragma unroll
        for (int t = 0; t < NT; ++t)
            *reinterpret_cast<float2*>(mine + 8 * t) =
                ROWS == 8 ? make_float2((acc[t][0] + acc[t][2]) * up, (acc[t][1] + acc[t][3]) * up)
                          : make_float2(acc[t][2 * h] * up, acc[t][2 * h + 1] * up);
        if (tq == 0) {
            ml[at * 2] = m[h];
            ml[at * 2 + 1] = l[h];
        }
    }
    __syncthreads();
    const int used = min(W, per_warp ? (c1 - c0 + per_warp - 1) / per_warp : 0);  // warps that had tiles
    constexpr int PARTS = W > ROWS ? W / ROWS : 1;  // warps of a row, each with a part of its columns
    for (int r = warp / PARTS; r < ROWS; r += W / PARTS) {
        const int rr = grp * ROWS + r;
        if (rr >= rows) return;
        // lane w has warp w's m and l
        const float2 own = lane < used ? *reinterpret_cast<const float2*>(ml + (lane * ROWS + r) * 2) : make_float2(-INFINITY, 0.f);
        float mm = own.x;
#pragma unroll
        for (int o = W / 2; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
        mm = __shfl_sync(0xffffffffu, mm, 0);
        const float mu = mm == -INFINITY ? 0.f : mm;
        const float fw = ex2(own.x - mu);
        float ll = 0.f;
        constexpr int D = HD / 32 / PARTS > 0 ? HD / 32 / PARTS : 1;
        float v[D] = {};
        const int d0 = (warp % PARTS) * (HD / PARTS) + lane;
#pragma unroll 8
        for (int w = 0; w < used; ++w) {
            const float f = __shfl_sync(0xffffffffu, fw, w);
            ll += f * __shfl_sync(0xffffffffu, own.y, w);
#pragma unroll
            for (int i = 0; i < D; ++i) v[i] += f * mo[(w * ROWS + r) * R::kPitch + d0 + 32 * i];
        }
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        const int tok = token_of(a, rr);
        const long long ob = tok * a.os + (long long)(kvh * a.group + rr - tok * a.group) * hd;
        const size_t pr = ((size_t)kvh * rows + rr) * a.nsplit + split;
#pragma unroll
        for (int i = 0; i < D; ++i) {
            const int p = d0 + 32 * i, d = (p & 7) * (HD / 8) + (p >> 3);
            if (d >= hd) continue;
            if (sh.whole()) o_store(a.o, a.type, ob + d, v[i] * inv);
            else a.part_o[pr * hd + d] = v[i];
        }
        if (lane == 0 && warp % PARTS == 0) {
            float* st = sh.whole() ? a.stats + ((size_t)kvh * rows + rr) * 2 : a.part_ml + pr * 2;
            st[0] = sh.whole() ? mu : mm;
            st[1] = sh.whole() ? inv : ll;
        }
    }
}

// A row's final m and 1 / l from its splits (or from the only one), by a warp.
__device__ __forceinline__ float2 row_stats(const AttnArgs& a, int kvh, int rr, const Shares& sh) {
    const int rows = a.n * a.group, lane = threadIdx.x & 31;
    if (sh.whole()) return *reinterpret_cast<const float2*>(a.stats + ((size_t)kvh * rows + rr) * 2);
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + ((size_t)kvh * rows + rr) * a.nsplit;
    const int n = sh.count();
    float2 x[kMaxSplit / 32];
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxSplit / 32; ++i) {
        x[i] = lane + 32 * i < n ? ml[lane + 32 * i] : make_float2(-INFINITY, 0.f);
        mm = fmaxf(mm, x[i].x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    const float mu = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int i = 0; i < kMaxSplit / 32; ++i) ll += ex2(x[i].x - mu) * x[i].y;
#pragma unroll
    for (int o = 16; o; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
    return make_float2(mu, ll == 0.f ? 0.f : 1.f / ll);
}

// After the splits: the first `joins` CTAs of a KV head join rows' splits, in their order (a warp per row); the
// others, with weights kept and few rows, add up the rows' weights from the stored scores (1024 keys a CTA).
__global__ void __launch_bounds__(256) kv8_join_kernel(const __grid_constant__ AttnArgs a, int joins) {
    __shared__ float2 st[kPromptRows];
    pdl_wait();
    pdl_trigger();
    const int hd = (int)a.c.head_dim, cap = (int)a.c.capacity, rows = a.n * a.group;
    const int lane = threadIdx.x & 31, kvh = blockIdx.y, past = *a.c.past;
    if ((int)blockIdx.x < joins) {
        const int rr = blockIdx.x * 8 + (threadIdx.x >> 5);
        if (rr >= rows) return;
        const Shares sh = shares_of(a, past, rr / a.unit);
        if (sh.whole()) return;
        const size_t pr = ((size_t)kvh * rows + rr) * a.nsplit;
        const float *ml = a.part_ml + pr * 2, *po = a.part_o + pr * hd;
        const int n = sh.count();
        // lane s has share s's (and s + 32's) m and l
        float2 own[kMaxSplit / 32];
        float mm = -INFINITY;
#pragma unroll
        for (int i = 0; i < kMaxSplit / 32; ++i) {
            own[i] = lane + 32 * i < n ? *reinterpret_cast<const float2*>(ml + 2 * (lane + 32 * i)) : make_float2(-INFINITY, 0.f);
            mm = fmaxf(mm, own[i].x);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
        const float mu = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int i = 0; i < kMaxSplit / 32; ++i) own[i].x = ex2(own[i].x - mu);
        float ll = 0.f, v[8] = {};
        // four columns of a share a lane and load; eight shares in flight (hd is a multiple of 16)
        auto add = [&](int s, int from, float f) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (4 * lane + 128 * i < hd) {
                    const float4 x = *reinterpret_cast<const float4*>(po + (size_t)(from + s) * hd + 4 * lane + 128 * i);
                    v[4 * i] += f * x.x;
                    v[4 * i + 1] += f * x.y;
                    v[4 * i + 2] += f * x.z;
                    v[4 * i + 3] += f * x.w;
                }
        };
#pragma unroll
        for (int i = 0; i < kMaxSplit / 32; ++i)
#pragma unroll 8
            for (int s = 0; s < min(32, n - 32 * i); ++s) {
                const float f = __shfl_sync(0xffffffffu, own[i].x, s);
                ll += f * __shfl_sync(0xffffffffu, own[i].y, s);
                add(s, 32 * i, f);
            }
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        const int tok = token_of(a, rr);
        const long long ob = tok * a.os + (long long)(kvh * a.group + rr - tok * a.group) * hd;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = 4 * lane + 128 * (i / 4) + i % 4;
            if (d < hd) o_store(a.o, a.type, ob + d, v[i] * inv);
        }
        if (lane == 0 && !a.scores) {  // (the weights' CTAs of few rows take their own)
            float* d = a.stats + ((size_t)kvh * rows + rr) * 2;
            d[0] = mu;
            d[1] = inv;
        }
        return;
    }
    const int keys = keys_of(past, a.n - 1, cap);
    const int key = ((int)blockIdx.x - joins) * 1024 + (int)threadIdx.x * 4;
    if (((int)blockIdx.x - joins) * 1024 >= keys) return;
    const float* t = a.scores + (size_t)kvh * ((rows + a.unit - 1) / a.unit * a.unit) * cap + key;
    float sum[4] = {};
    for (int r0 = 0; r0 < rows; r0 += 8) {
        float4 x[8];  // loaded before the statistics that they wait for
#pragma unroll
        for (int r = 0; r < 8; ++r)  // a row that sees none of the four keys may not have stored them
            x[r] = r0 + r < rows && key < keys_of(past, token_of(a, r0 + r), cap)
                       ? *reinterpret_cast<const float4*>(t + (size_t)(r0 + r) * cap)
                       : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (r0 == 0) {
            for (int r = threadIdx.x >> 5; r < rows; r += 8) {
                const float2 y = row_stats(a, kvh, r, shares_of(a, past, r / a.unit));
                if (lane == 0) st[r] = y;
            }
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (r0 + r >= rows) continue;
            const float mr = st[r0 + r].x, ir = st[r0 + r].y;
            const float v[4] = {x[r].x, x[r].y, x[r].z, x[r].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)  // (a row that is not a number spoils the keys that it sees, no others)
                if (v[e] != -INFINITY) sum[e] += ex2(v[e] - mr) * ir;
        }
    }
    if (key >= keys) return;
    float* w = a.weight + (size_t)kvh * cap + key;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (key + e < keys) w[e] = key + e < past ? w[e] + sum[e] : sum[e];
}


// Shares of few rows' keys at least, so that a warp's sums go over 1024 keys at most (see kChainKeys): one token of 96
// heads x 128 in fp32 over 120000 rows is 9e-7 off and takes 549 us (8.3e-6 and 686 in one share, 7500 keys a warp).
size_t rows_least_shares(const neon_kv8_t& c) {
    const size_t keys = (size_t)kChainKeys * (c.head_dim <= 128 ? RowTile<128, 8>::kWarps : RowTile<256, 8>::kWarps);
    return std::min<size_t>(kMaxSplit, (c.capacity + keys - 1) / keys);
}

// The plan of a call, from what the host knows of it (not how many rows the cache holds).
struct Plan {
    bool prompt;
    int unit, nsplit;
    size_t stats, part_o, part_ml, sums, scores, qt, qfactor, bytes;  // offsets into the workspace
};
Plan plan_of(const neon_kv8_t& c, size_t n, size_t n_head, int type) {
    Plan p{};
    const size_t rows = n * (n_head / c.n_kv_head), H = c.n_kv_head, hd = c.head_dim;
    p.prompt = rows > (size_t)kPromptRows;
    p.unit = p.prompt ? prompt_unit((int)hd) : rows > 8 && type != NEON_GGML_F32 ? 16 : 8;
    const size_t units = H * ((rows + p.unit - 1) / p.unit);
    // shares of the keys: as many as fill the SMs once, and for prompts at least 512 rows each (a share per 128 rows
    // takes 24.5 us for 300 tokens where this takes 20.1; per 2048 rows, 54 for 40 tokens behind 2000 where this
    // takes 26). Few rows take a block per warp at least (min_tiles: 512 rows, 256 above head_dim 128); the limit here
    // only has to leave room for that (one token over 4000 rows of 8 heads x 128 takes 12.6 us; with a limit of one
    // per 512 rows, seven shares of 18 blocks for 16 warps, 14.3), and is 1 for short caches, which then need no join.
    const size_t most = p.prompt ? c.capacity / 512 : c.capacity < 1024 ? 1 : c.capacity / 256;
    p.nsplit = (int)std::max<size_t>(1, std::min<size_t>({(size_t)kMaxSplit, kSms / units, most}));
    if (!p.prompt) p.nsplit = (int)std::max<size_t>(p.nsplit, rows_least_shares(c));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at = (at + bytes + 1023) & ~(size_t)1023;
        return o;
    };
    p.stats = take(H * rows * 2 * sizeof(float));
    p.part_o = take(p.nsplit > 1 ? H * rows * p.nsplit * hd * sizeof(float) : 0);
    p.part_ml = take(p.nsplit > 1 ? H * rows * p.nsplit * 2 * sizeof(float) : 0);
    p.sums = take(p.prompt && c.capacity > (size_t)kChainKeys ? units * p.unit * p.nsplit * hd * sizeof(float) : 0);
    // what only weights need comes last
    p.scores = take(p.prompt ? 0 : H * ((rows + p.unit - 1) / p.unit) * p.unit * c.capacity * sizeof(float));
    const size_t padded = (rows + 255) / 256 * 256;
    p.qfactor = take(p.prompt ? H * padded * sizeof(float) : 0);
    p.qt = take(p.prompt ? prompt_query_bytes(c, rows, type) : 0);
    p.bytes = at + 1024;  // the caller's 16-byte alignment is rounded up
    return p;
}

template <int ROWS>
int launch_rows(AttnArgs& a, cudaStream_t st) {
    const int hd = (int)a.c.head_dim;
    auto k = hd == 64    ? kv8_rows_kernel<64, true, ROWS>
             : hd < 64   ? kv8_rows_kernel<64, false, ROWS>
             : hd == 128 ? kv8_rows_kernel<128, true, ROWS>
             : hd < 128  ? kv8_rows_kernel<128, false, ROWS>
             : hd == 256 ? kv8_rows_kernel<256, true, ROWS>
                         : kv8_rows_kernel<256, false, ROWS>;
    const int smem = hd <= 64    ? RowTile<64, ROWS>::kSmem
                     : hd <= 128 ? RowTile<128, ROWS>::kSmem
                                 : RowTile<256, ROWS>::kSmem;
    const int warps = hd <= 128 ? RowTile<128, ROWS>::kWarps : RowTile<256, ROWS>::kWarps;
    // a tile per warp before another CTA joins (one token over 512 and 1500 rows takes 7.7 and 11.4 us; with no
    // least share 7.6 and 11.3, with four tiles a warp 7.6 and 15.1: the fewer shares to join are free)
    a.min_tiles = warps;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return neon_internal::cuda_error(e, "cudaFuncSetAttribute(kv8_rows_kernel)");
    const unsigned groups = (unsigned)((a.n * a.group + ROWS - 1) / ROWS);
    return launch("kv8_rows_kernel", k, dim3((unsigned)a.nsplit, a.c.n_kv_head, groups), warps * 32, (size_t)smem, st, 1, a);
}

}  // namespace

size_t kv8_attention_workspace(const neon_kv8_t& c, size_t n, size_t n_head, bool weights) {
    // Fewer tokens may take more shares, but rows * shares is at most kSms units' rows, or `few` (plan_of).
    const size_t rows = n * (n_head / c.n_kv_head), H = c.n_kv_head;
    const size_t unit = rows > (size_t)kPromptRows ? prompt_unit((int)c.head_dim) : 16;
    const size_t padded = (rows + 255) / 256 * 256;
    const size_t few = H * ((std::min<size_t>(rows, kPromptRows) + 15) / 16 * 16) * rows_least_shares(c);
    const size_t parts = std::max(kSms * unit, few) * (c.head_dim + 2) * sizeof(float);
    const size_t sums = rows > (size_t)kPromptRows && c.capacity > (size_t)kChainKeys
                            ? std::max(kSms * unit, H * ((rows + unit - 1) / unit * unit)) * c.head_dim * sizeof(float)
                            : 0;
    const size_t scores = H * ((std::min<size_t>(rows, kPromptRows) + 15) / 16 * 16) * c.capacity * sizeof(float);
    return H * rows * 2 * sizeof(float) + parts + sums + 10 * 1024 +
           (weights ? H * padded * sizeof(float) + prompt_query_bytes(c, rows, NEON_GGML_F32) + scores : 0);
}

int kv8_attention(const neon_kv8_t& c, const void* q, size_t qs, void* o, size_t os, size_t n, size_t n_head,
                  float scale, int type, float* weight, void* ws, int device, cudaStream_t st) {
    unsigned* err = neon_internal::device_error_word(device);
    if (!err) return NEON_ERR_CUDA;
    const Plan p = plan_of(c, n, n_head, type);
    unsigned char* base = (unsigned char*)(((uintptr_t)ws + 1023) & ~(uintptr_t)1023);
    AttnArgs a{};
    a.c = c;
    a.q = q;
    a.o = o;
    a.qs = (long long)qs;
    a.os = (long long)os;
    a.n = (int)n;
    a.n_head = (int)n_head;
    a.group = (int)(n_head / c.n_kv_head);
    a.type = type;
    a.scale = scale * kLog2e;
    a.weight = weight;
    a.nsplit = p.nsplit;
    a.unit = p.unit;
    a.stats = (float*)(base + p.stats);
    a.part_o = (float*)(base + p.part_o);
    a.part_ml = (float*)(base + p.part_ml);
    a.sums = (float4*)(base + p.sums);
    a.qt = base + p.qt;
    a.qfactor = (float*)(base + p.qfactor);
    a.err = err;
    const size_t rows = n * a.group;
    int rc;
    if (p.prompt) {
        a.tile_shift = prompt_tile_shift();
        a.min_tiles = 8;  // (300 tokens of 16 / 8 heads take 21.5 us with 8 and with 1, 21.7 with 32)
        rc = launch_prompt(a, st);
    } else {
        a.tile_shift = 5;
        if (weight) a.scores = (float*)(base + p.scores);
        rc = p.unit == 8 ? launch_rows<8>(a, st) : launch_rows<16>(a, st);
    }
    const unsigned joins = a.nsplit > 1 ? (unsigned)((rows + 7) / 8) : 0;
    const unsigned sums = a.scores ? (c.capacity + 1023) / 1024 : 0;
    if (!rc && joins + sums)
        rc = launch("kv8_join_kernel", kv8_join_kernel, dim3(joins + sums, c.n_kv_head), 256, 0, st, 1, a, (int)joins);
    if (!rc && weight && p.prompt) rc = launch_prompt_weights(a, st);
    return rc;
}

}  // namespace longctx

using namespace longctx;
using neon_internal::error;

namespace {
int check_heads(const neon_kv8_t* c, size_t n, size_t n_head) {
    int rc = kv8_check(c);
    if (rc) return rc;
    if (n_head == 0 || n_head % c->n_kv_head) return error(NEON_ERR_INVALID, "kv8: n_head must be a multiple of n_kv_head");
    if (n_head / c->n_kv_head > 64) return error(NEON_ERR_UNSUPPORTED, "kv8: more than 64 query heads per KV head");
    if (n > c->capacity) return error(NEON_ERR_INVALID, "kv8: more tokens than the cache's capacity");
    if (n * (n_head / c->n_kv_head) > (1u << 26)) return error(NEON_ERR_UNSUPPORTED, "kv8: more than 2^26 query rows per KV head");
    return NEON_OK;
}
}  // namespace

extern "C" {

int neon_cuda_kv8_attention_workspace(const neon_kv8_t* cache, size_t n, size_t n_head, size_t* bytes) {
    if (!bytes) return error(NEON_ERR_INVALID, "null bytes");
    int rc = check_heads(cache, n, n_head);
    if (rc) return rc;
    *bytes = kv8_attention_workspace(*cache, n, n_head, true);
    return NEON_OK;
}

int neon_cuda_kv8_attention(const neon_kv8_t* cache, const void* dQ, size_t q_stride, void* dO, size_t o_stride,
                            size_t n, size_t n_head, float scale, int type, float* d_weight, void* workspace,
                            size_t workspace_bytes, void* stream) {
    int rc = kv8_check_buffers(cache);
    if (!rc) rc = check_heads(cache, n, n_head);
    if (rc) return rc;
    const size_t eb = type_bytes(type);
    if (!eb) return error(NEON_ERR_UNSUPPORTED, "kv8: type must be F32, F16 or BF16");
    if (n == 0) return NEON_OK;
    if (!dQ || !dO || !workspace) return error(NEON_ERR_INVALID, "kv8: null Q, O or workspace");
    if (dQ == dO) return error(NEON_ERR_INVALID, "kv8: Q and O must not be the same buffer");
    const size_t row = n_head * cache->head_dim;
    if (n > 1 && (q_stride < row || o_stride < row)) return error(NEON_ERR_INVALID, "kv8: stride smaller than the heads");
    if (!aligned(dQ, eb) || !aligned(dO, eb) || !aligned(d_weight, 4) || !aligned(workspace, 16))
        return error(NEON_ERR_INVALID, "kv8: buffer not aligned (workspace: 16 bytes)");
    if (!std::isfinite(scale)) return error(NEON_ERR_INVALID, "kv8: scale must be finite");
    const size_t need = kv8_attention_workspace(*cache, n, n_head, true);
    if (workspace_bytes < need)
        return error(NEON_ERR_INVALID, "kv8: workspace below neon_cuda_kv8_attention_workspace() = " + std::to_string(need));
    if (scale == 0.f) scale = 1.f / std::sqrt((float)cache->head_dim);
    if (!apart(dQ, q_stride * eb, row * eb, dO, o_stride * eb, row * eb, n))
        return error(NEON_ERR_INVALID, "kv8: Q and O must not overlap");
    OnDevice dev(cache->k);
    if (dev.rc) return dev.rc;
    return kv8_attention(*cache, dQ, q_stride, dO, o_stride, n, n_head, scale, type, d_weight, workspace, dev.device,
                         (cudaStream_t)stream);
}

}  // extern "C"
