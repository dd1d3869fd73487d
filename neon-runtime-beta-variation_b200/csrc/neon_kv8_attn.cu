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

// p (at most 1, times s_v over the largest s_v so far) is multiplied by 2^14
// before its split: hi stays below fp16's 65504, and lo keeps values down to
// 2^-38 of the row's largest.
constexpr float kPUp = 16384.f, kPDown = 1.f / 16384.f;

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------------------
// Eight rows of one KV head over a share of the cache. The MMA's 16 rows hold
// the eight rows' hi terms and below them their lo terms, so the split costs
// no extra products: a row's score is the sum of its two halves, and its
// output likewise. Each warp streams its own tiles of 32 rows (a block of the
// cache: K and V codes as two bulk copies) through its own ring in shared
// memory, with no barrier between the warps until their results are merged.
// The order of the summed dimension is free, so each lane reads whole 16-byte
// pieces of a K row and the query fragments are laid out to match; of V, lane
// group g takes columns [g HD / 8, (g + 1) HD / 8) of four rows.
// ---------------------------------------------------------------------------
constexpr int kRowWarps = 8;
constexpr int kRowThreads = kRowWarps * 32;

template <int HD>
struct RowTile {
    static constexpr int kStages = HD <= 64 ? 4 : HD <= 128 ? 3 : 1;
    static constexpr int kStageBytes = 2 * 32 * HD;
    static constexpr int kRingBytes = kRowWarps * kStages * kStageBytes;
    static constexpr int kMergeBytes = kRowWarps * 8 * (HD + 2) * 4;
    static constexpr int kSmem = (kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes) + 128 + kRowWarps * kStages * 8;
};

template <int HD>
__global__ void __launch_bounds__(kRowThreads, 1) kv8_rows_kernel(const __grid_constant__ AttnArgs a) {
    using R = RowTile<HD>;
    constexpr int KS = HD / 16;   // k-steps of the score product
    constexpr int NT = HD / 8;    // column tiles of the output
    extern __shared__ __align__(128) unsigned char smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (R::kRingBytes > R::kMergeBytes ? R::kRingBytes : R::kMergeBytes));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
    const int hd = (int)a.c.head_dim, cap = (int)a.c.capacity;
    const int split = blockIdx.x, kvh = blockIdx.y, grp = blockIdx.z, rows = a.n * a.group;
    unsigned char* ring = smem + warp * R::kStages * R::kStageBytes;
    uint64_t* bar = bars + warp * R::kStages;
    if (lane == 0) {
        for (int s = 0; s < R::kStages; ++s) bar_init(&bar[s], 1);
        bar_init_fence();
    }
    __syncwarp();
    pdl_wait();
    pdl_trigger();

    // the keys of the group's rows, and this warp's share of them in tiles
    const int past = *a.c.past;
    const int row = grp * 8 + g, tok = row / a.group;
    const int limit = row < rows ? keys_of(past, tok, cap) : 0;
    const Shares sh = shares_of(a, past, grp);
    if (split >= sh.active) return;
    const int c0 = split * sh.per, c1 = min(c0 + sh.per, sh.tiles);
    const int per_warp = (c1 - c0 + kRowWarps - 1) / kRowWarps;
    const int w0 = min(c0 + warp * per_warp, c1), w1 = min(w0 + per_warp, c1);

    const int8_t* kc = a.c.k + (size_t)kvh * cap * hd;
    const int8_t* vc = a.c.v + (size_t)kvh * cap * hd;
    const float* ksc = a.c.k_scale + (size_t)kvh * (cap >> 5);
    const float* vsc = a.c.v_scale + (size_t)kvh * (cap >> 5);
    const uint32_t bytes = 32u * hd;
    auto issue = [&](int tile) {
        const int s = (tile - w0) % R::kStages;
        unsigned char* d = ring + s * R::kStageBytes;
        bar_expect(&bar[s], 2 * bytes);
        bulk_load(d, kc + (size_t)tile * bytes, bytes, &bar[s]);
        bulk_load(d + 32 * HD, vc + (size_t)tile * bytes, bytes, &bar[s]);
    };
    if (lane == 0)
        for (int t = w0; t < min(w0 + R::kStages, w1); ++t) issue(t);

    // Query fragments: lane (g, tq) holds values tq HD / 4 + 4 s .. + 3 of row g for step s, times
    // 2^-e so that the row's largest is near 2^7 (its lo terms then stay normal halves).
    uint32_t qf[KS][4];
    float factor;
    {
        float x[HD / 4];
        float mx = 0.f;
        const long long base = (long long)tok * a.qs + (long long)(kvh * a.group + row % a.group) * hd;
#pragma unroll
        for (int i = 0; i < HD / 4; ++i) {
            const int d = tq * (HD / 4) + i;
            x[i] = row < rows && d < hd ? q_value(a.q, a.type, base + d) : 0.f;
            mx = fmaxf(mx, fabsf(x[i]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = mx > 0.f && !isinf(mx) ? 7 - ilogbf(mx) : 0;
        factor = ldexpf(a.scale, -e);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            split2(ldexpf(x[4 * s], e), ldexpf(x[4 * s + 1], e), qf[s][0], qf[s][1]);
            split2(ldexpf(x[4 * s + 2], e), ldexpf(x[4 * s + 3], e), qf[s][2], qf[s][3]);
        }
    }

    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    float m = -INFINITY, l = 0.f, vref = 0.f;
    float my_ks = 0.f, my_vs = 0.f;  // the scales of 32 tiles, one per lane
    bool ok = true;
    for (int tile = w0; tile < w1; ++tile) {
        const int it = tile - w0, s = it % R::kStages;
        if ((it & 31) == 0) {
            const int b = tile + lane;
            my_ks = b < w1 ? ksc[b] : 0.f;
            my_vs = b < w1 ? vsc[b] : 0.f;
        }
        const float ks = __shfl_sync(0xffffffffu, my_ks, it & 31), vs = __shfl_sync(0xffffffffu, my_vs, it & 31);
        ok = ok && bar_wait(&bar[s], (uint32_t)((it / R::kStages) & 1), a.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const unsigned char* kt = ring + s * R::kStageBytes;
        const unsigned char* vt = kt + 32 * HD;

        // scores of 32 keys: key 8 j + g of column tile j
        float sc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[j][e] = 0.f;
            const unsigned char* kr = kt + (8 * j + g) * hd + tq * (HD / 4);
#pragma unroll
            for (int p = 0; p < HD / 64; ++p) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (tq * (HD / 4) + 16 * p < hd) w = *reinterpret_cast<const uint4*>(kr + 16 * p);
                const uint32_t u[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
                for (int i = 0; i < 4; ++i) mma16816(sc[j], qf[4 * p + i], codes_lo(u[i]), codes_hi(u[i]));
            }
        }
        // online softmax of row g: the lane has keys 8 j + 2 tq and + 1
        const float kf = factor * ks;
        float t[4][2], mt = m;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = tile * 32 + 8 * j + 2 * tq + e;
                t[j][e] = key < limit ? (sc[j][e] + sc[j][e + 2]) * kf : -INFINITY;
                mt = fmaxf(mt, t[j][e]);
            }
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        const float mu = mt == -INFINITY ? 0.f : mt;
        const float down = ex2(m - mu);
        float vdown = 1.f;
        if (vs > vref) {
            vdown = vref / vs;
            vref = vs;
        }
        const float vr = vs == 0.f ? 0.f : vs / vref * kPUp;
        l *= down;
        m = mt;
        if (__any_sync(0xffffffffu, down * vdown != 1.f)) {
            const float f = down * vdown;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][e] *= f;
        }
        uint32_t pf[2][4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int j = 2 * k + hf;
                const bool on0 = t[j][0] != -INFINITY, on1 = t[j][1] != -INFINITY;
                const float p0 = ex2(t[j][0] - mu), p1 = ex2(t[j][1] - mu);
                l += p0 + p1;
                split2(on0 ? p0 * vr : 0.f, on1 ? p1 * vr : 0.f, pf[k][2 * hf], pf[k][2 * hf + 1]);
            }
        }
        // o += p V: lane (g, tq) reads columns g HD / 8 .. of rows 16 k + 2 tq, + 1, + 8, + 9
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const unsigned char* vrow = vt + (16 * k + 2 * tq) * hd + g * (HD / 8);
            constexpr int W = HD / 32;  // words of a lane's columns
            uint32_t w[4][W];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned char* src = vrow + ((r & 1) + 8 * (r >> 1)) * hd;
                if constexpr (W == 2) {
                    uint2 v = make_uint2(0, 0);
                    if (g * 8 < hd) v = *reinterpret_cast<const uint2*>(src);
                    w[r][0] = v.x ^ 0x80808080u;
                    w[r][1] = v.y ^ 0x80808080u;
                } else {
#pragma unroll
                    for (int p = 0; p < W / 4; ++p) {
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
            for (int i = 0; i < W; ++i) {
                // bytes (r0 c0, r1 c0, r0 c1, r1 c1) and (.. c2, .. c3) of both row pairs
                const uint32_t a01 = __byte_perm(w[0][i], w[1][i], 0x5140), a23 = __byte_perm(w[0][i], w[1][i], 0x7362);
                const uint32_t b01 = __byte_perm(w[2][i], w[3][i], 0x5140), b23 = __byte_perm(w[2][i], w[3][i], 0x7362);
                mma16816(acc[4 * i], pf[k], codes_lo(a01), codes_lo(b01));
                mma16816(acc[4 * i + 1], pf[k], codes_hi(a01), codes_hi(b01));
                mma16816(acc[4 * i + 2], pf[k], codes_lo(a23), codes_lo(b23));
                mma16816(acc[4 * i + 3], pf[k], codes_hi(a23), codes_hi(b23));
            }
        }
        __syncwarp();
        if (lane == 0 && tile + R::kStages < w1) issue(tile + R::kStages);
    }
    if (!ok)  // let this warp's copies end (each wait bounded) before shared memory is reused
        for (int s = 0; s < R::kStages; ++s) bar_wait(&bar[s], 0, a.err);

    // merge the warps: o (times s_v), m, l of each row
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    __syncthreads();
    float* mo = reinterpret_cast<float*>(smem);             // [warps][8][HD]
    float* ml = mo + kRowWarps * 8 * HD;                     // [warps][8][2]
    const float up = vref * kPDown;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float* o = mo + (warp * 8 + g) * HD;
        o[2 * tq * (HD / 8) + t] = (acc[t][0] + acc[t][2]) * up;
        o[(2 * tq + 1) * (HD / 8) + t] = (acc[t][1] + acc[t][3]) * up;
    }
    if (tq == 0) {
        ml[(warp * 8 + g) * 2] = m;
        ml[(warp * 8 + g) * 2 + 1] = l;
    }
    __syncthreads();
    for (int r = warp; r < 8; r += kRowWarps) {
        const int rr = grp * 8 + r;
        if (rr >= rows) continue;
        float mm = -INFINITY;
        for (int w = 0; w < kRowWarps; ++w) mm = fmaxf(mm, ml[(w * 8 + r) * 2]);
        const float mu = mm == -INFINITY ? 0.f : mm;
        float f[kRowWarps], ll = 0.f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) {
            f[w] = ex2(ml[(w * 8 + r) * 2] - mu);
            ll += f[w] * ml[(w * 8 + r) * 2 + 1];
        }
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        const long long ob = (long long)(rr / a.group) * a.os + (long long)(kvh * a.group + rr % a.group) * hd;
        const size_t pr = ((size_t)kvh * rows + rr) * a.nsplit + split;
        for (int d = lane; d < hd; d += 32) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) v += f[w] * mo[(w * 8 + r) * HD + d];
            if (sh.active == 1) o_store(a.o, a.type, ob + d, v * inv);
            else a.part_o[pr * hd + d] = v;
        }
        if (lane == 0) {
            float* st = sh.active == 1 ? a.stats + ((size_t)kvh * rows + rr) * 2 : a.part_ml + pr * 2;
            st[0] = sh.active == 1 ? mu : mm;
            st[1] = sh.active == 1 ? inv : ll;
        }
    }
}

// Joins a row's splits, in their order. One warp per row.
__global__ void __launch_bounds__(128) kv8_join_kernel(const __grid_constant__ AttnArgs a) {
    pdl_wait();
    pdl_trigger();
    const int hd = (int)a.c.head_dim, rows = a.n * a.group;
    const int lane = threadIdx.x & 31;
    const int rr = blockIdx.x * 4 + (threadIdx.x >> 5), kvh = blockIdx.y;
    if (rr >= rows) return;
    const Shares sh = shares_of(a, *a.c.past, rr / a.unit);
    if (sh.active == 1) return;
    const size_t pr = ((size_t)kvh * rows + rr) * a.nsplit;
    const float *ml = a.part_ml + pr * 2, *po = a.part_o + pr * hd;
    float mm = -INFINITY;
    for (int s = lane; s < sh.active; s += 32) mm = fmaxf(mm, ml[2 * s]);
#pragma unroll
    for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    const float mu = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, v[8] = {};
#pragma unroll 4
    for (int s = 0; s < sh.active; ++s) {
        const float f = ex2(ml[2 * s] - mu);
        ll += f * ml[2 * s + 1];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd) v[i] += f * po[(size_t)s * hd + lane + 32 * i];
    }
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    const long long ob = (long long)(rr / a.group) * a.os + (long long)(kvh * a.group + rr % a.group) * hd;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < hd) o_store(a.o, a.type, ob + lane + 32 * i, v[i] * inv);
    if (lane == 0) {
        float* st = a.stats + ((size_t)kvh * rows + rr) * 2;
        st[0] = mu;
        st[1] = inv;
    }
}

// ---------------------------------------------------------------------------
// The rows' weights: a warp owns 32 cached rows (one block), keeps their codes
// as fragments, goes through the query rows in groups of eight and sums each
// column of p. Needs the rows' final m and 1 / l.
// ---------------------------------------------------------------------------
template <int HD>
__global__ void __launch_bounds__(256, 1) kv8_weight_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int KS = HD / 16;
    __shared__ uint32_t qs[KS][32][4];
    __shared__ float qfac[8], qm[8], qi[8];
    __shared__ int qlim[8];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
    const int hd = (int)a.c.head_dim, cap = (int)a.c.capacity, kvh = blockIdx.y, rows = a.n * a.group;
    const int past = *a.c.past;
    const int keys = keys_of(past, a.n - 1, cap);
    if ((int)blockIdx.x * 256 >= keys) return;
    const int tile = blockIdx.x * 8 + warp;  // this warp's block
    const bool on = tile * 32 < keys;
    uint32_t kf[4][KS][2];
    float ks = 0.f;
    if (on) {
        ks = a.c.k_scale[(size_t)kvh * (cap >> 5) + tile];
        const int8_t* kc = a.c.k + ((size_t)kvh * cap + 32 * tile) * hd;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int p = 0; p < HD / 64; ++p) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (tq * (HD / 4) + 16 * p < hd)
                    w = *reinterpret_cast<const uint4*>(kc + (8 * j + g) * hd + tq * (HD / 4) + 16 * p);
                const uint32_t u[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    kf[j][4 * p + i][0] = codes_lo(u[i]);
                    kf[j][4 * p + i][1] = codes_hi(u[i]);
                }
            }
    }
    float sum[4][2] = {};
    // the first row that sees any key of the CTA
    const int first = (int)max(0LL, min((long long)rows, ((long long)blockIdx.x * 256 - past) * a.group)) / 8;
    for (int grp = first; grp * 8 < rows; ++grp) {
        __syncthreads();
        if (warp == 0) {
            const int row = grp * 8 + g, tok = row / a.group;
            float x[HD / 4];
            float mx = 0.f;
            const long long base = (long long)tok * a.qs + (long long)(kvh * a.group + row % a.group) * hd;
#pragma unroll
            for (int i = 0; i < HD / 4; ++i) {
                const int d = tq * (HD / 4) + i;
                x[i] = row < rows && d < hd ? q_value(a.q, a.type, base + d) : 0.f;
                mx = fmaxf(mx, fabsf(x[i]));
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const int e = mx > 0.f && !isinf(mx) ? 7 - ilogbf(mx) : 0;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                split2(ldexpf(x[4 * s], e), ldexpf(x[4 * s + 1], e), qs[s][lane][0], qs[s][lane][1]);
                split2(ldexpf(x[4 * s + 2], e), ldexpf(x[4 * s + 3], e), qs[s][lane][2], qs[s][lane][3]);
            }
            if (tq == 0) {
                const float* st = a.stats + ((size_t)kvh * rows + min(row, rows - 1)) * 2;
                qfac[g] = ldexpf(a.scale, -e);
                qm[g] = st[0];
                qi[g] = row < rows ? st[1] : 0.f;
                qlim[g] = row < rows ? keys_of(past, tok, cap) : 0;
            }
        }
        __syncthreads();
        if (!on) continue;
        const float fac = qfac[g] * ks, mrow = qm[g], irow = qi[g];
        const int lim = qlim[g];
        float sc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[j][e] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint32_t q[4] = {qs[s][lane][0], qs[s][lane][1], qs[s][lane][2], qs[s][lane][3]};
#pragma unroll
            for (int j = 0; j < 4; ++j) mma16816(sc[j], q, kf[j][s][0], kf[j][s][1]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = tile * 32 + 8 * j + 2 * tq + e;
                if (key < lim) sum[j][e] += ex2((sc[j][e] + sc[j][e + 2]) * fac - mrow) * irow;
            }
    }
    if (!on) return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float v = sum[j][e];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            const int key = tile * 32 + 8 * j + 2 * tq + e;
            if (g == 0 && key < keys) {
                float* w = a.weight + (size_t)kvh * cap + key;
                *w = key < past ? *w + v : v;
            }
        }
}

constexpr int kMaxSplit = 64;
constexpr int kPromptRows = 32;  // query rows of a KV head from which on the prompt kernel takes them

// The plan of a call, from what the host knows of it (not how many rows the cache holds).
struct Plan {
    bool prompt;
    int unit, nsplit;
    size_t stats, part_o, part_ml, qt, qfactor, bytes;  // offsets into the workspace
};
Plan plan_of(const neon_kv8_t& c, size_t n, size_t n_head, int type) {
    Plan p{};
    const size_t rows = n * (n_head / c.n_kv_head), H = c.n_kv_head, hd = c.head_dim;
    p.prompt = rows > (size_t)kPromptRows;
    p.unit = p.prompt ? prompt_unit((int)hd) : 8;
    const size_t units = H * ((rows + p.unit - 1) / p.unit);
    // shares of the keys: as many as fill the SMs once
    p.nsplit = (int)std::max<size_t>(1, std::min<size_t>({(size_t)kMaxSplit, 148 / units, (size_t)c.capacity / 512}));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at = (at + bytes + 1023) & ~(size_t)1023;
        return o;
    };
    p.stats = take(H * rows * 2 * sizeof(float));
    p.part_o = take(p.nsplit > 1 ? H * rows * p.nsplit * hd * sizeof(float) : 0);
    p.part_ml = take(p.nsplit > 1 ? H * rows * p.nsplit * 2 * sizeof(float) : 0);
    const size_t padded = (rows + 255) / 256 * 256;
    p.qfactor = take(p.prompt ? H * padded * sizeof(float) : 0);
    p.qt = take(p.prompt ? prompt_query_bytes(c, rows, type) : 0);
    p.bytes = at + 1024;  // the caller's 16-byte alignment is rounded up
    return p;
}

}  // namespace

size_t kv8_attention_workspace(const neon_kv8_t& c, size_t n, size_t n_head) {
    // Fewer tokens may take more shares, but rows * shares is at most 148 units' rows (plan_of).
    const size_t rows = n * (n_head / c.n_kv_head), H = c.n_kv_head;
    const size_t unit = rows > (size_t)kPromptRows ? std::max(8, prompt_unit((int)c.head_dim)) : 8;
    const size_t padded = (rows + 255) / 256 * 256;
    return H * rows * 2 * sizeof(float) + 148 * unit * (c.head_dim + 2) * sizeof(float) + H * padded * sizeof(float) +
           prompt_query_bytes(c, rows, NEON_GGML_F32) + 8 * 1024;
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
    a.qt = base + p.qt;
    a.qfactor = (float*)(base + p.qfactor);
    a.err = err;
    const size_t rows = n * a.group;
    const int hd = (int)c.head_dim;
    int rc;
    if (p.prompt) {
        a.tile_keys = prompt_tile_keys();
        a.min_tiles = 8;
        rc = launch_prompt(a, st);
    } else {
        a.tile_keys = 32;
        a.min_tiles = 2 * kRowWarps;  // two tiles per warp
        auto rows_kernel = hd <= 64 ? kv8_rows_kernel<64> : hd <= 128 ? kv8_rows_kernel<128> : kv8_rows_kernel<256>;
        const int smem = hd <= 64 ? RowTile<64>::kSmem : hd <= 128 ? RowTile<128>::kSmem : RowTile<256>::kSmem;
        cudaError_t e = cudaFuncSetAttribute(rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return neon_internal::cuda_error(e, "cudaFuncSetAttribute(kv8_rows_kernel)");
        rc = launch("kv8_rows_kernel", rows_kernel, dim3((unsigned)a.nsplit, c.n_kv_head, (unsigned)((rows + 7) / 8)),
                    kRowThreads, (size_t)smem, st, 1, a);
    }
    if (!rc && a.nsplit > 1)
        rc = launch("kv8_join_kernel", kv8_join_kernel, dim3((unsigned)((rows + 3) / 4), c.n_kv_head), 128, 0, st, 1, a);
    if (!rc && weight && p.prompt) {
        rc = launch_prompt_weights(a, st);
    } else if (!rc && weight) {
        auto wk = hd <= 64 ? kv8_weight_kernel<64> : hd <= 128 ? kv8_weight_kernel<128> : kv8_weight_kernel<256>;
        rc = launch("kv8_weight_kernel", wk, dim3((c.capacity + 255) / 256, c.n_kv_head), 256, 0, st, 1, a);
    }
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
    return NEON_OK;
}
}  // namespace

extern "C" {

int neon_cuda_kv8_attention_workspace(const neon_kv8_t* cache, size_t n, size_t n_head, size_t* bytes) {
    if (!bytes) return error(NEON_ERR_INVALID, "null bytes");
    int rc = check_heads(cache, n, n_head);
    if (rc) return rc;
    *bytes = kv8_attention_workspace(*cache, n, n_head);
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
    const size_t row = n_head * cache->head_dim;
    if (n > 1 && (q_stride < row || o_stride < row)) return error(NEON_ERR_INVALID, "kv8: stride smaller than the heads");
    if (!aligned(dQ, eb) || !aligned(dO, eb) || !aligned(d_weight, 4) || !aligned(workspace, 16))
        return error(NEON_ERR_INVALID, "kv8: buffer not aligned (workspace: 16 bytes)");
    if (!std::isfinite(scale)) return error(NEON_ERR_INVALID, "kv8: scale must be finite");
    const size_t need = kv8_attention_workspace(*cache, n, n_head);
    if (workspace_bytes < need)
        return error(NEON_ERR_INVALID, "kv8: workspace below neon_cuda_kv8_attention_workspace() = " + std::to_string(need));
    if (scale == 0.f) scale = 1.f / std::sqrt((float)cache->head_dim);
    OnDevice dev(cache->k);
    if (dev.rc) return dev.rc;
    return kv8_attention(*cache, dQ, q_stride, dO, o_stride, n, n_head, scale, type, d_weight, workspace, dev.device,
                         (cudaStream_t)stream);
}

}  // extern "C"
