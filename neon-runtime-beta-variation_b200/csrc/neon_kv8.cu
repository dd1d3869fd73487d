// neon_kv8.cu -- the KV cache in 8 bits: append, read and eviction
// (neon_cuda_kv8_append / _read / _evict). The attention over it is in
// neon_kv8_attn.cu.
//
// A block is 32 rows of one KV head: codes c = rint(x / s), s = amax / 127. A
// code is the nearest integer to the exact quotient: the quotient is first
// taken with the reciprocal of s, which settles it unless it is near a tie.
// There the remainder e = x - r s, which one FMA gives exactly (r is at most one off the nearest integer, so e is a
// multiple of the smaller ulp and below s), moves r by one where |e| > s / 2
// and to the even side where |e| = s / 2. So the codes do not depend on how a
// quotient is rounded, and a block's codes are a function of its rows.
#include "neon_longctx.cuh"
#include "neon_kv8.h"

#include <algorithm>

namespace longctx {

int kv8_check(const neon_kv8_t* c) {
    using neon_internal::error;
    if (!c) return error(NEON_ERR_INVALID, "null cache");
    if (c->n_kv_head == 0 || c->n_kv_head > 16384) return error(NEON_ERR_INVALID, "kv8: n_kv_head must be 1 to 16384");
    if (c->head_dim < 16 || c->head_dim % 16 || c->head_dim > 256)
        return error(NEON_ERR_UNSUPPORTED, "kv8: head_dim must be a multiple of 16, from 16 to 256");
    if (c->capacity == 0 || c->capacity % NEON_KV8_BLOCK || c->capacity > (1u << 30))
        return error(NEON_ERR_INVALID, "kv8: capacity must be a multiple of 32, from 32 to 2^30");
    return NEON_OK;
}

int kv8_check_buffers(const neon_kv8_t* c) {
    using neon_internal::error;
    int rc = kv8_check(c);
    if (rc) return rc;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->tail || !c->tail_block || !c->past)
        return error(NEON_ERR_INVALID, "kv8: null buffer");
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->tail, 16))
        return error(NEON_ERR_INVALID, "kv8: codes and tail must be 16-byte aligned");
    if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(c->tail_block, 4) || !aligned(c->past, 4))
        return error(NEON_ERR_INVALID, "kv8: buffer not aligned to its type");
    return NEON_OK;
}

namespace {

constexpr float kTiny = 127.f * 1.17549435e-38f;  // 127 * FLT_MIN

// A block's scale from its largest magnitude (as bits).
__device__ __forceinline__ float block_scale(unsigned top) {
    const float amax = __uint_as_float(top);
    return top >= 0x7f800000u ? __int_as_float(0x7fffffff) : amax >= kTiny ? __fdiv_rn(amax, 127.f) : 0.f;
}
// The largest of a CTA of four warps.
__device__ __forceinline__ unsigned block_top(unsigned m, unsigned* red) {
    const unsigned top = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    return max(max(red[0], red[1]), max(red[2], red[3]));
}

// The nearest integer to x / s, ties to even, from x times the reciprocal: as is where that is clear of a tie
// (the product is off by less than 2^-15 of an integer), else by the exact remainder.
__device__ __forceinline__ int quantise_exact(float x, float s, float inv) {
    float r = rintf(__fmul_rn(x, inv));
    const float e = __fmaf_rn(-r, s, x);  // exact
    const float e2 = 2.f * fabsf(e);
    if (e2 > s || (e2 == s && ((int)r & 1))) r += e > 0.f ? 1.f : -1.f;
    return (int)r;
}
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, which the low byte then holds
constexpr float kNearTie = 0.4999f;

// Four quotients (as two pairs) as rounded codes; far: how far one is from its code.
__device__ __forceinline__ uint32_t round4(uint64_t y01, uint64_t y23, float& far) {
    const uint64_t up = pair(kMagic, kMagic), down = pair(-kMagic, -kMagic), minus = pair(-1.f, -1.f);
    const uint64_t t01 = add2(y01, up), t23 = add2(y23, up);
    float d0, d1, d2, d3, t0, t1, t2, t3;
    unpair(fma2(add2(t01, down), minus, y01), d0, d1);
    unpair(fma2(add2(t23, down), minus, y23), d2, d3);
    far = fmaxf(fmaxf(fabsf(d0), fabsf(d1)), fmaxf(fabsf(d2), fabsf(d3)));
    unpair(t01, t0, t1);
    unpair(t23, t2, t3);
    return __byte_perm(__byte_perm(__float_as_uint(t0), __float_as_uint(t1), 0x0040),
                       __byte_perm(__float_as_uint(t2), __float_as_uint(t3), 0x0040), 0x5410);
}
__device__ __noinline__ uint32_t exact4(float4 x, float s, float inv) {
    return (uint32_t)(quantise_exact(x.x, s, inv) & 255) | (uint32_t)(quantise_exact(x.y, s, inv) & 255) << 8 |
           (uint32_t)(quantise_exact(x.z, s, inv) & 255) << 16 | (uint32_t)(quantise_exact(x.w, s, inv) & 255) << 24;
}
// Four values as four codes.
__device__ __forceinline__ uint32_t quantise4(const float (&x)[4], float s, float inv) {
    const uint64_t i2 = pair(inv, inv);
    float far;
    const uint32_t c = round4(mul2(pair(x[0], x[1]), i2), mul2(pair(x[2], x[3]), i2), far);
    return far > kNearTie ? exact4(make_float4(x[0], x[1], x[2], x[3]), s, inv) : c;
}

// Four codes as floats: 0x4b0000uu is 2^23 + u, with u = code + 128 (an int-to-float conversion has a quarter of
// the rate).
__device__ __forceinline__ void code_pairs(uint32_t w, uint64_t& c01, uint64_t& c23) {
    const uint32_t u = w ^ 0x80808080u;
    const uint64_t bias = pair(-8388736.f, -8388736.f);
    c01 = add2(pair(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7541))), bias);
    c23 = add2(pair(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7542)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7543))), bias);
}
__device__ __forceinline__ void code_values(uint32_t w, float s, float (&x)[4]) {
    uint64_t c01, c23;
    code_pairs(w, c01, c23);
    unpair(mul2(c01, pair(s, s)), x[0], x[1]);
    unpair(mul2(c23, pair(s, s)), x[2], x[3]);
}
// Magnitudes as bit patterns order like numbers, and what is not finite is at or above 0x7f800000.
__device__ __forceinline__ unsigned magnitude(const float (&x)[4]) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
    return m;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// A CTA of four warps per block, head and K or V; the first CTA of a head
// takes its first block and then its last one, the only two that touch the
// tail. A thread has 8 pieces of 4 values at head_dim 128, all loaded before
// the first is used. 8191 rows of 8 heads x 128 in bf16 take 19 us where their
// bytes are 8: loads, the block's largest value, then the rounding, one after
// the other in each CTA; one token's is a launch and its latency (4.4 us).

struct AppendArgs {
    neon_kv8_t c;
    const void *k, *v;
    long long ks, vs;
    int n;
    bool vec;
    unsigned* dropped;  // the device's word for rows beyond the capacity
};
constexpr int kAppThreads = 128;

// HD: the head dimension, known to the compiler, or 0 (then P covers a.c.head_dim).
template <typename T, int HD, int P = HD ? HD / 16 : 16>
__global__ void __launch_bounds__(kAppThreads) kv8_append_kernel(const __grid_constant__ AppendArgs a) {
    __shared__ unsigned red[2][kAppThreads / 32];
    pdl_wait();
    pdl_trigger();
    const int hd = HD ? HD : (int)a.c.head_dim, cap = (int)a.c.capacity, H = (int)a.c.n_kv_head;
    const int h = blockIdx.y, which = blockIdx.z, tid = threadIdx.x;
    const int past = *a.c.past;
    if (past < 0 || (long long)past + a.n > cap) {
        if (tid == 0 && h == 0 && which == 0 && blockIdx.x == 0) *a.dropped = 1u;
        if (past < 0 || past >= cap) return;
    }
    const int end = (int)min((long long)past + a.n, (long long)cap);
    const int b0 = past >> 5, b1 = (end - 1) >> 5, r0 = past & 31;
    int b = b0 + (int)blockIdx.x;
    if (blockIdx.x > 0 && b >= b1) return;
    const T* src = (const T*)(which ? a.v : a.k);
    const long long ss = which ? a.vs : a.ks;
    int8_t* codes = (which ? a.c.v : a.c.k) + (size_t)h * cap * hd;
    float* scales = (which ? a.c.v_scale : a.c.k_scale) + (size_t)h * (cap >> 5);
    const size_t slot_floats = (size_t)H * 32 * hd;
    float* tail = a.c.tail + ((size_t)which * 2 * H + h) * 32 * hd;  // slot s at + s * slot_floats
    int* tag = a.c.tail_block + ((size_t)which * H + h) * 2;

    // The slots of the first and the last block (the head's first CTA alone
    // looks at them): the first block's rows are kept if it has earlier rows,
    // the last block's always, in the other slot.
    int slot0 = -1, slot1 = -1;
    bool known = false;
    if (blockIdx.x == 0) {
        const int g0 = tag[0], g1 = tag[1];
        if (r0) {
            known = g0 == b0 || g1 == b0;
            slot0 = g0 == b0 ? 0 : g1 == b0 ? 1 : g0 == b0 - 1 ? 1 : 0;
            if (b1 > b0) slot1 = 1 - slot0;
        } else if (b1 == b0) {
            slot0 = g0 == b0 - 1 ? 1 : 0;
        } else {
            slot1 = g0 == b1 - 1 ? 1 : 0;
        }
        __syncthreads();  // every thread has read the tags
        if (tid < 2) {
            const int g = tid ? g1 : g0;
            // blocks that this call writes are no longer what an older slot holds
            const int now = tid == slot0 ? b0 : tid == slot1 ? b1 : g >= b0 && g <= b1 ? -1 : g;
            if (now != g) tag[tid] = now;
        }
    }
    for (int pass = 0;; ++pass) {
        const int rows = min(32, end - 32 * b);  // rows that the block holds after this call
        const int old = b == b0 ? r0 : 0;        // of them, rows from before
        const int slot = blockIdx.x == 0 ? (b == b0 ? slot0 : slot1) : -1;
        float* keep = slot >= 0 ? tail + slot * slot_floats : nullptr;
        uint32_t* bc = reinterpret_cast<uint32_t*>(codes + (size_t)b * 32 * hd);
        const int per = hd / 4;  // pieces of a row
        if (old == 0 && rows == 32 && a.vec && !keep) {  // a new, whole block: most of a prompt's
            Vec4<T> w[P];
            const T* q = src + (32LL * b - past) * ss + (long long)h * hd;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int p = i * kAppThreads + tid, r = p / per;
                if (r < 32) w[i].load(q + r * ss + (p - r * per) * 4);
            }
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < P; ++i)
                if ((i * kAppThreads + tid) / per < 32) {
                    const float x[4] = {to_f(w[i].t[0]), to_f(w[i].t[1]), to_f(w[i].t[2]), to_f(w[i].t[3])};
                    m = max(m, magnitude(x));
                }
            const float s = block_scale(block_top(m, red[pass & 1])), inv = __fdiv_rn(1.f, s);
#pragma unroll
            for (int i = 0; i < P; ++i)
                if ((i * kAppThreads + tid) / per < 32) {
                    const float x[4] = {to_f(w[i].t[0]), to_f(w[i].t[1]), to_f(w[i].t[2]), to_f(w[i].t[3])};
                    bc[i * kAppThreads + tid] = s > 0.f ? quantise4(x, s, inv) : 0u;
                }
            if (tid == 0) scales[b] = s;
            if (blockIdx.x > 0 || b == b1) break;
            b = b1;
            known = false;
            continue;
        }
        Vec4<T> w[P];
        int row[P];
        // the new rows' loads alone first, all in flight together
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int p = i * kAppThreads + tid;
            row[i] = p / per;
            if (row[i] >= old && row[i] < rows) {
                const T* q = src + (32LL * b + row[i] - past) * ss + (long long)h * hd + (p - row[i] * per) * 4;
                if (a.vec) {
                    w[i].load(q);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[i].t[e] = q[e];
                }
            }
        }
        const float before = old && !known ? scales[b] : 0.f;
        float x[P][4];
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int p = i * kAppThreads + tid;
            if (row[i] >= old && row[i] < rows) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = to_f(w[i].t[e]);
            } else if (row[i] < old && known) {
                const float4 v = *reinterpret_cast<const float4*>(keep + 4 * p);
                x[i][0] = v.x; x[i][1] = v.y; x[i][2] = v.z; x[i][3] = v.w;
            } else if (row[i] < old) {
                code_values(bc[p], before, x[i]);
            } else {
                x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
            }
            m = max(m, magnitude(x[i]));
        }
        const float s = block_scale(block_top(m, red[pass & 1]));
        const float inv = __fdiv_rn(1.f, s);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int p = i * kAppThreads + tid;
            if (row[i] < rows) {
                bc[p] = s > 0.f ? quantise4(x[i], s, inv) : 0u;  // an empty block, or NaN: 0
                if (keep && (row[i] >= old || !known))
                    *reinterpret_cast<float4*>(keep + 4 * p) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
            }
        }
        if (tid == 0) scales[b] = s;
        if (blockIdx.x > 0 || b == b1) break;
        b = b1;
        known = false;
    }
}

using AppendKernel = void (*)(AppendArgs);
template <typename T>
AppendKernel append_kernel_for(int hd) {
    return hd == 64 ? kv8_append_kernel<T, 64> : hd == 128 ? kv8_append_kernel<T, 128> : kv8_append_kernel<T, 0>;
}

// ---------------------------------------------------------------------------
// read
// ---------------------------------------------------------------------------
// A piece of four codes per lane, so that a warp's loads and stores are whole
// lines; eight pieces in flight a thread. The fp32 rows that it writes bound it:
// 32768 rows of 8 heads x 128 take 60 us (5.6 TB/s).
constexpr int kReadThreads = 256, kReadRows = 64;  // rows of a CTA

__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(const __grid_constant__ neon_kv8_t c, int row0, int n,
                                                                float* k_out, float* v_out) {
    pdl_wait();
    pdl_trigger();
    const int hd = (int)c.head_dim, cap = (int)c.capacity, H = (int)c.n_kv_head, h = blockIdx.y, which = blockIdx.z;
    float* out = which ? v_out : k_out;
    if (!out) return;
    const int first = row0 + (int)blockIdx.x * kReadRows, rows = min(kReadRows, row0 + n - first);
    const uint32_t* codes = reinterpret_cast<const uint32_t*>((which ? c.v : c.k) + ((size_t)h * cap + first) * hd);
    const float* scales = (which ? c.v_scale : c.k_scale) + (size_t)h * (cap >> 5);
    float* to = out + ((size_t)(first - row0) * H + h) * hd;
    const int per = hd / 4, total = rows * per;
    const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0;  // (a caller's buffer is aligned to its floats only)
    constexpr int U = 8;
    for (int i0 = threadIdx.x; i0 < total; i0 += kReadThreads * U) {
        uint32_t q[U];
        float s[U];
        int r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kReadThreads;
            r[u] = i / per;
            if (i < total) {
                q[u] = codes[i];
                s[u] = scales[(first + r[u]) >> 5];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kReadThreads;
            if (i >= total) continue;
            float* o = to + (size_t)r[u] * H * hd + (i - r[u] * per) * 4;
            float x[4];
            code_values(q[u], s[u], x);
            if (vec) {
                *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
                o[0] = x[0]; o[1] = x[1]; o[2] = x[2]; o[3] = x[3];
            }
        }
    }
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
// Two launches. The first finds each head's kept rows: a cluster of CTAs per
// head takes the m-th largest weight by four rounds of 8-bit radix counts
// (weights as ordered bit patterns, so the selection is exact), then writes
// the rows above it, and the lowest rows equal to it, in order: each warp owns
// a range of rows, and its place is a prefix sum over the warps. The second
// gathers: one CTA per new block, head and K or V.

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelHeld = 16;  // weights that a thread holds (16384 rows of a head and CTA); any others are read again

// A weight as an unsigned number of the same order; every NaN is the largest.
__device__ __forceinline__ unsigned order_bits(float w) {
    const unsigned u = __float_as_uint(w + 0.f);  // -0 as 0
    if (w != w) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ unsigned remote_u32(const unsigned* p, int rank) {
    unsigned a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct SelectArgs {
    const int* past;
    const float* w;  // [H][cap]
    int cap, keep, sink, recent;
    int* kept;       // [H][keep]
};

// CL: CTAs of a head, a cluster. One takes 1024 rows in 8 us and 8192 in 13.6 where eight, with their barriers, take
// 11 and 13.7; eight take 131071 rows in 27 us. Loads, counts in shared memory and barriers bound it, in rounds.
template <int CL>
__global__ void __launch_bounds__(kSelThreads) kv8_select_kernel(const __grid_constant__ SelectArgs a) {
    __shared__ unsigned hist[2][256];
    __shared__ unsigned sum[256];
    __shared__ unsigned counts[2 * kSelWarps];       // rows above / equal of this CTA's warps
    __shared__ unsigned all[2 * kSelWarps * CL];
    __shared__ unsigned found[3];
    pdl_wait();
    pdl_trigger();
    const int h = blockIdx.x / CL, rank = blockIdx.x % CL;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int len = min(max(*a.past, 0), a.cap);
    int* kept = a.kept + (size_t)h * a.keep;
    if (len <= a.keep) {  // everything stays (the whole cluster takes this path)
        for (int i = rank * kSelThreads + tid; i < a.keep; i += CL * kSelThreads) kept[i] = i < len ? i : -1;
        return;
    }
    const float* w = a.w + (size_t)h * a.cap;
    const int lo = a.sink, hi = len - a.recent, m = a.keep - a.sink - a.recent;  // hi - lo > m >= 0
    for (int i = rank * kSelThreads + tid; i < a.sink; i += CL * kSelThreads) kept[i] = i;
    for (int i = rank * kSelThreads + tid; i < a.recent; i += CL * kSelThreads) kept[a.keep - a.recent + i] = hi + i;
    if (m == 0) return;

    // Held weights are this warp's: rows s0 + 32 j + lane.
    const int nw = CL * kSelWarps, gw = rank * kSelWarps + warp;
    const int span = ((hi - lo + nw - 1) / nw + 31) & ~31;
    const int s0 = min(lo + gw * span, hi), s1 = min(s0 + span, hi);
    unsigned held[kSelHeld];
#pragma unroll
    for (int j = 0; j < kSelHeld; ++j) held[j] = s0 + 32 * j + lane < s1 ? order_bits(w[s0 + 32 * j + lane]) : 0u;
    // f(row, its ordered weight, whether it is one of the warp's), for whole warps and in row order
    auto each = [&](auto f) {
#pragma unroll
        for (int j = 0; j < kSelHeld; ++j)
            if (s0 + 32 * j < s1) f(s0 + 32 * j + lane, held[j], s0 + 32 * j + lane < s1);
        for (int i0 = s0 + 32 * kSelHeld; i0 < s1; i0 += 32) {
            const bool on = i0 + lane < s1;
            f(i0 + lane, on ? order_bits(w[i0 + lane]) : 0u, on);
        }
    };

    // the m-th largest, eight bits a round
    unsigned prefix = 0, left = (unsigned)m;
    bool closed = false;  // every row from the threshold on stays: no need to look further down
    for (int round = 0; round < 4 && !closed; ++round) {
        const int shift = 24 - 8 * round;
        unsigned* hs = hist[round & 1];
        for (int i = tid; i < 256; i += kSelThreads) hs[i] = 0;
        __syncthreads();
        each([&](int, unsigned u, bool on) {
            if (on && (round == 0 || (u >> (shift + 8)) == prefix)) atomicAdd(&hs[(u >> shift) & 255], 1u);
        });
        if (CL > 1) cluster_barrier();
        else __syncthreads();
        // bin 255 - tid and the bins above it, over the cluster
        if (tid < 256) {
            unsigned c = 0;
#pragma unroll
            for (int r = 0; r < CL; ++r) c += CL > 1 ? remote_u32(&hs[255 - tid], r) : hs[255 - tid];
            unsigned s = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned v = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += v;
            }
            sum[tid] = s;
        }
        __syncthreads();
        if (tid < 256) {
            unsigned base = 0;
            for (int k = 0; k < warp; ++k) base += sum[k * 32 + 31];
            const unsigned upto = base + sum[tid], above = tid == 0 ? 0u : (lane ? base + sum[tid - 1] : base);
            if (above < left && left <= upto) {
                found[0] = 255u - tid;
                found[1] = left - above;
                found[2] = upto - above;
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | found[0];
        left = found[1];
        closed = left == found[2];
        if (closed) prefix <<= shift;
    }
    // rows above T stay, and the first `left` rows equal to it; closed: rows from T on
    const unsigned T = prefix;
    if (closed) left = 0;

    unsigned above = 0, equal = 0;
    each([&](int, unsigned u, bool on) {
        above += on && (u > T || (closed && u == T));
        equal += on && u == T && !closed;
    });
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) {
        counts[warp] = above;
        counts[kSelWarps + warp] = equal;
    }
    if (CL > 1) cluster_barrier();
    else __syncthreads();
    for (int i = tid; i < 2 * nw; i += kSelThreads) {
        const int r = i / (2 * kSelWarps);
        all[i] = CL > 1 ? remote_u32(&counts[i % (2 * kSelWarps)], r) : counts[i];
    }
    __syncthreads();
    unsigned before = 0, ties = 0;  // of the warps before this one
    for (int k = lane; k < gw; k += 32) {
        before += all[(k / kSelWarps) * 2 * kSelWarps + k % kSelWarps];
        ties += all[(k / kSelWarps) * 2 * kSelWarps + kSelWarps + k % kSelWarps];
    }
    before = __reduce_add_sync(0xffffffffu, before);
    ties = __reduce_add_sync(0xffffffffu, ties);
    each([&](int i, unsigned u, bool on) {
        const bool up = on && (u > T || (closed && u == T)), eq = on && u == T && !closed;
        const unsigned bu = __ballot_sync(0xffffffffu, up), be = __ballot_sync(0xffffffffu, eq);
        const unsigned mask = (1u << lane) - 1u;
        const unsigned t = ties + __popc(be & mask);  // equal rows before this one
        if (up || (eq && t < left)) kept[a.sink + before + __popc(bu & mask) + min(t, left)] = i;
        before += __popc(bu);
        ties += __popc(be);
    });
    if (CL > 1) cluster_barrier();  // no CTA leaves while another reads its counts
}

struct GatherArgs {
    neon_kv8_t src, dst;
    const float* w;
    float* wd;
    const int* kept;
    int keep;
    int pairs, half, rotate;
    RopeTurns turns;
};
constexpr int kGatherThreads = 128;

// A CTA of four warps per new block, head and K or V, in pieces of four codes, P a thread. The largest magnitude is
// a row's largest code times its scale. HD as for the append. 32768 of 131071 rows of 8 heads x 128 take 55 us where
// their bytes are 20: rows of 128 bytes from anywhere, and the rounding. CTAs that take several blocks, the next
// one's rows loaded while one is quantised, are no faster (an eviction of 148 to 158 us against 146).
template <int HD, int P = HD ? HD / 16 : 16>
__global__ void __launch_bounds__(kGatherThreads) kv8_gather_kernel(const __grid_constant__ GatherArgs a) {
    extern __shared__ __align__(16) float rowbuf[];  // with rotation: the block's rows
    __shared__ unsigned red[kGatherThreads / 32];
    __shared__ int from[32];
    __shared__ float fs[32];
    pdl_wait();
    pdl_trigger();
    const int hd = HD ? HD : (int)a.src.head_dim, H = (int)a.src.n_kv_head, cap = (int)a.src.capacity, dcap = (int)a.dst.capacity;
    const int b = blockIdx.x, h = blockIdx.y, which = blockIdx.z, tid = threadIdx.x;
    const float* ssc = (which ? a.src.v_scale : a.src.k_scale) + (size_t)h * (cap >> 5);
    const int r_ = tid < 32 && 32 * b + tid < a.keep ? a.kept[(size_t)h * a.keep + 32 * b + tid] : -1;  // -1 behind the last
    if (b == 0) {
        const int m = min(min(max(*a.src.past, 0), cap), a.keep);
        if (tid < 2) a.dst.tail_block[((size_t)which * H + h) * 2 + tid] = -1;
        if (h == 0 && which == 0 && tid == 0) *a.dst.past = m;
    }
    if (tid < 32) {
        from[tid] = r_;
        if (r_ >= 0) {
            fs[tid] = ssc[r_ >> 5];
            if (which == 0 && a.wd) a.wd[(size_t)h * dcap + 32 * b + tid] = a.w[(size_t)h * cap + r_];
        }
    }
    __syncthreads();
    int rows = 32;
    if (from[31] < 0) {  // the last block
        rows = 0;
        while (rows < 32 && from[rows] >= 0) ++rows;
        if (rows == 0) return;
    }
    // kept rows ascend: the last one in place means that all of the block's are
    const bool stay = from[rows - 1] == 32 * b + rows - 1;
    const int8_t* sc = (which ? a.src.v : a.src.k) + (size_t)h * cap * hd;
    uint32_t* dc = reinterpret_cast<uint32_t*>((which ? a.dst.v : a.dst.k) + ((size_t)h * dcap + 32 * b) * hd);
    float* dsc = (which ? a.dst.v_scale : a.dst.k_scale) + (size_t)h * (dcap >> 5);
    const int per = hd / 4;
    uint32_t q[P];
    int row[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int p = i * kGatherThreads + tid;
        row[i] = p / per;
        q[i] = 0;
        if (row[i] < rows) q[i] = *reinterpret_cast<const uint32_t*>(sc + (size_t)from[row[i]] * hd + (p - row[i] * per) * 4);
    }
    if (stay) {
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (row[i] < rows) dc[i * kGatherThreads + tid] = q[i];
        if (tid == 0) dsc[b] = fs[0];
        return;
    }
    const bool turned = a.rotate && which == 0;
    unsigned m = 0;
    if (!turned) {
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (row[i] < rows) {
                const uint32_t u = __vabs4(q[i]);  // (codes are -127 .. 127)
                const unsigned top = max(max(u & 255, (u >> 8) & 255), max((u >> 16) & 255, u >> 24));
                m = max(m, __float_as_uint(__fmul_rn((float)top, fs[row[i]])));  // scales are not negative
            }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (row[i] < rows) {
                float x[4];
                code_values(q[i], fs[row[i]], x);
                *reinterpret_cast<float4*>(rowbuf + 4 * (i * kGatherThreads + tid)) = make_float4(x[0], x[1], x[2], x[3]);
            }
        __syncthreads();
        for (int i = tid; i < rows * a.pairs; i += kGatherThreads) {
            const int r = i / a.pairs, p = i - r * a.pairs;
            const int delta = 32 * b + r - from[r];
            if (delta == 0) continue;
            const float2 c = turn(a.turns.f[p], delta);
            float* u = rowbuf + r * hd + (a.half ? p : 2 * p);
            float* v = u + (a.half ? a.pairs : 1);
            const float x0 = *u, x1 = *v;
            *u = __fmaf_rn(x0, c.x, -__fmul_rn(x1, c.y));
            *v = __fmaf_rn(x0, c.y, __fmul_rn(x1, c.x));
        }
        __syncthreads();
        for (int i = tid; i < rows * hd; i += kGatherThreads) m = max(m, __float_as_uint(rowbuf[i]) & 0x7fffffffu);
    }
    const float sn = block_scale(block_top(m, red));
    const float inv = __fdiv_rn(1.f, sn);
#pragma unroll
    for (int i = 0; i < P; ++i) {
        if (row[i] >= rows) continue;
        const int p = i * kGatherThreads + tid;
        if (turned) {
            const float4 v = *reinterpret_cast<const float4*>(rowbuf + 4 * p);
            const float x[4] = {v.x, v.y, v.z, v.w};
            dc[p] = sn > 0.f ? quantise4(x, sn, inv) : 0u;
        } else {
            // a code times the row's scale over the new one; the value itself only where that is near a tie
            const float s = fs[row[i]], rho = __fmul_rn(s, inv);
            uint64_t c01, c23;
            code_pairs(q[i], c01, c23);
            float far;
            uint32_t c = round4(mul2(c01, pair(rho, rho)), mul2(c23, pair(rho, rho)), far);
            if (far > kNearTie) {
                float x[4];
                code_values(q[i], s, x);
                c = exact4(make_float4(x[0], x[1], x[2], x[3]), sn, inv);
            }
            dc[p] = sn > 0.f ? c : 0u;
        }
    }
    if (tid == 0) dsc[b] = sn;
}

// Rows from row0 to the end of row1's block as zeros: a CTA per block, head and K or V. The first block keeps its scale
// where it has earlier rows, and the slot of the tail that holds it those rows; no slot holds one of the others any more.
__global__ void __launch_bounds__(128) kv8_clear_kernel(const __grid_constant__ neon_kv8_t c, float* w, int row0, int row1) {
    pdl_wait();
    pdl_trigger();
    const int hd = (int)c.head_dim, cap = (int)c.capacity, H = (int)c.n_kv_head, h = blockIdx.y, which = blockIdx.z, tid = threadIdx.x;
    const int b0 = row0 >> 5, b = b0 + (int)blockIdx.x, r0 = b == b0 ? row0 & 31 : 0;
    uint4* codes = reinterpret_cast<uint4*>((which ? c.v : c.k) + ((size_t)h * cap + 32 * b) * hd);
    for (int i = r0 * hd / 16 + tid; i < 2 * hd; i += 128) codes[i] = make_uint4(0, 0, 0, 0);
    if (r0 == 0 && tid == 0) (which ? c.v_scale : c.k_scale)[(size_t)h * (cap >> 5) + b] = 0.f;
    if (which == 0 && w && tid < 32 && tid >= r0 && 32 * b + tid < row1) w[(size_t)h * cap + 32 * b + tid] = 0.f;
    if (blockIdx.x) return;
    int* tag = c.tail_block + ((size_t)which * H + h) * 2;
    for (int s = 0; s < 2; ++s) {
        const int g = tag[s];
        if (r0 && g == b0) {
            float4* t = reinterpret_cast<float4*>(c.tail + (((size_t)which * 2 + s) * H + h) * 32 * hd);
            for (int i = r0 * hd / 4 + tid; i < 8 * hd; i += 128) t[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        } else if (g >= b0 && g <= (row1 - 1) >> 5) {
            __syncthreads();  // every thread has read the tag
            if (tid == 0) tag[s] = -1;
        }
    }
}

}  // namespace

int kv8_clear(const neon_kv8_t& c, float* w, size_t row0, size_t row1, cudaStream_t st) {
    if (row0 >= row1) return NEON_OK;
    const unsigned blocks = (unsigned)((row1 + 31) / 32 - row0 / 32);
    return launch("kv8_clear_kernel", kv8_clear_kernel, dim3(blocks, c.n_kv_head, 2), 128, 0, st, 1, c, w, (int)row0, (int)row1);
}

int kv8_append(const neon_kv8_t& c, const void* k, size_t ks, const void* v, size_t vs, size_t n, int type, int device,
               cudaStream_t st) {
    unsigned* dropped = neon_internal::device_rows_word(device);
    if (!dropped) return NEON_ERR_CUDA;
    const size_t eb = type_bytes(type);
    AppendArgs a{};
    a.c = c;
    a.k = k;
    a.v = v;
    a.ks = (long long)ks;
    a.vs = (long long)vs;
    a.n = (int)n;
    a.vec = aligned(k, 4 * eb) && aligned(v, 4 * eb) && ks % 4 == 0 && vs % 4 == 0;
    a.dropped = dropped;
    AppendKernel kern = type == NEON_GGML_F32   ? append_kernel_for<float>((int)c.head_dim)
                        : type == NEON_GGML_F16 ? append_kernel_for<__half>((int)c.head_dim)
                                                : append_kernel_for<__nv_bfloat16>((int)c.head_dim);
    // rows past .. past + n - 1 touch at most (n + 62) / 32 blocks; the first CTA takes two of them
    const unsigned blocks = (unsigned)std::max<size_t>(1, (n + 62) / 32 - 1);
    return launch("kv8_append_kernel", kern, dim3(blocks, c.n_kv_head, 2), kAppThreads, 0, st, 1, a);
}

int kv8_move(const neon_kv8_t& src, const float* w, const neon_kv8_t& dst, float* wd, size_t keep, const neon_rope_t* rope,
             const int32_t* kept, cudaStream_t st) {
    GatherArgs g{};
    g.src = src;
    g.dst = dst;
    g.w = w;
    g.wd = wd;
    g.kept = kept;
    g.keep = (int)keep;
    if (rope) {
        g.rotate = 1;
        g.pairs = (int)rope->n_dims / 2;
        g.half = rope->layout == NEON_ROPE_HALF;
        const int rc = rope_turns(*rope, &g.turns);
        if (rc) return rc;
    }
    const int hd = (int)src.head_dim;
    auto kern = hd == 64 ? kv8_gather_kernel<64> : hd == 128 ? kv8_gather_kernel<128> : kv8_gather_kernel<0>;
    return launch("kv8_gather_kernel", kern, dim3((unsigned)((keep + 31) / 32), src.n_kv_head, 2), kGatherThreads,
                  rope ? (size_t)32 * hd * sizeof(float) : 0, st, 1, g);
}

int kv8_evict(const neon_kv8_t& src, const float* w, const neon_kv8_t& dst, float* wd, size_t keep, size_t sink,
              size_t recent, const neon_rope_t* rope, int32_t* kept, cudaStream_t st) {
    RopeTurns turns;
    if (rope)  // (nothing is launched for a rotation that is not one)
        if (const int bad = rope_turns(*rope, &turns)) return bad;
    SelectArgs s{src.past, w, (int)src.capacity, (int)keep, (int)sink, (int)recent, kept};
    const bool one = src.capacity <= kSelThreads * kSelHeld;  // a CTA holds all of a head's weights
    int rc = one ? launch("kv8_select_kernel", kv8_select_kernel<1>, dim3(src.n_kv_head), kSelThreads, 0, st, 1, s)
                 : launch("kv8_select_kernel", kv8_select_kernel<8>, dim3(src.n_kv_head * 8), kSelThreads, 0, st, 8, s);
    return rc ? rc : kv8_move(src, w, dst, wd, keep, rope, kept, st);
}

}  // namespace longctx

using namespace longctx;
using neon_internal::error;

extern "C" {

int neon_cuda_kv8_append(const neon_kv8_t* cache, const void* dK, size_t k_stride, const void* dV, size_t v_stride,
                         size_t n, int type, void* stream) {
    int rc = kv8_check_buffers(cache);
    if (rc) return rc;
    const size_t eb = type_bytes(type);
    if (!eb) return error(NEON_ERR_UNSUPPORTED, "kv8: type must be F32, F16 or BF16");
    if (n == 0) return NEON_OK;
    if (!dK || !dV) return error(NEON_ERR_INVALID, "kv8: null K or V");
    if (n > cache->capacity) return error(NEON_ERR_INVALID, "kv8: more tokens than the cache's capacity");
    const size_t row = (size_t)cache->n_kv_head * cache->head_dim;
    if (n > 1 && (k_stride < row || v_stride < row)) return error(NEON_ERR_INVALID, "kv8: stride smaller than the heads");
    if (!aligned(dK, eb) || !aligned(dV, eb)) return error(NEON_ERR_INVALID, "kv8: buffer not aligned to its type");
    OnDevice dev(cache->k);
    if (dev.rc) return dev.rc;
    return kv8_append(*cache, dK, k_stride, dV, v_stride, n, type, dev.device, (cudaStream_t)stream);
}

int neon_cuda_kv8_read(const neon_kv8_t* cache, size_t row0, size_t n, float* dK_out, float* dV_out, void* stream) {
    int rc = kv8_check_buffers(cache);
    if (rc) return rc;
    if (row0 > cache->capacity || n > cache->capacity - row0) return error(NEON_ERR_INVALID, "kv8: rows out of range");
    if (!aligned(dK_out, 4) || !aligned(dV_out, 4)) return error(NEON_ERR_INVALID, "kv8: buffer not aligned to its type");
    if (n == 0 || (!dK_out && !dV_out)) return NEON_OK;
    OnDevice dev(cache->k);
    if (dev.rc) return dev.rc;
    if (neon_internal::device_sms(dev.device) < 0) return NEON_ERR_CUDA;
    return launch("kv8_read_kernel", kv8_read_kernel, dim3((unsigned)((n + kReadRows - 1) / kReadRows), cache->n_kv_head, 2),
                  kReadThreads, 0, (cudaStream_t)stream, 1, *cache, (int)row0, (int)n, dK_out, dV_out);
}

int neon_cuda_kv8_evict(const neon_kv8_t* src, const float* d_weight, const neon_kv8_t* dst, float* d_weight_dst,
                        size_t keep, size_t sink, size_t recent, const neon_rope_t* rope, int32_t* d_kept,
                        void* stream) {
    int rc = kv8_check_buffers(src);
    if (!rc) rc = kv8_check_buffers(dst);
    if (!rc && rope) rc = rope_check(rope, src->head_dim);
    if (rc) return rc;
    if (!d_weight || !d_weight_dst || !d_kept) return error(NEON_ERR_INVALID, "kv8: null weights or kept rows");
    if (!aligned(d_weight, 4) || !aligned(d_weight_dst, 4) || !aligned(d_kept, 4))
        return error(NEON_ERR_INVALID, "kv8: buffer not aligned to its type");
    if (src->n_kv_head != dst->n_kv_head || src->head_dim != dst->head_dim)
        return error(NEON_ERR_INVALID, "kv8: the caches' heads differ");
    if (keep == 0 || keep > dst->capacity) return error(NEON_ERR_INVALID, "kv8: keep must be 1 to the new cache's capacity");
    if (sink > keep || recent > keep - sink) return error(NEON_ERR_INVALID, "kv8: sink + recent above keep");
    const auto codes = [](const neon_kv8_t* c) { return (size_t)c->n_kv_head * c->capacity * c->head_dim; };
    const size_t H = src->n_kv_head, from = codes(src), to = codes(dst), tags = H * 4 * sizeof(int32_t);
    // (the tails are neither read nor written: one may serve both caches, as long as one of them is in use)
    const Range in[] = {{src->k, from}, {src->v, from}, {src->k_scale, from / src->head_dim / 8}, {src->v_scale, from / src->head_dim / 8},
                        {src->tail_block, tags}, {src->past, sizeof(int32_t)}, {d_weight, H * src->capacity * sizeof(float)}};
    const Range out[] = {{dst->k, to}, {dst->v, to}, {dst->k_scale, to / dst->head_dim / 8}, {dst->v_scale, to / dst->head_dim / 8},
                         {dst->tail_block, tags}, {dst->past, sizeof(int32_t)}, {d_weight_dst, H * dst->capacity * sizeof(float)},
                         {d_kept, H * keep * sizeof(int32_t)}};
    for (const Range& o : out) {
        for (const Range& i : in)
            if (o.meets(i)) return error(NEON_ERR_INVALID, "kv8: eviction needs separate buffers");
        for (const Range& p : out)
            if (&p != &o && o.meets(p)) return error(NEON_ERR_INVALID, "kv8: eviction needs separate buffers");
    }
    OnDevice dev(src->k);
    if (dev.rc) return dev.rc;
    if (neon_internal::device_sms(dev.device) < 0) return NEON_ERR_CUDA;
    return kv8_evict(*src, d_weight, *dst, d_weight_dst, keep, sink, recent, rope, d_kept, (cudaStream_t)stream);
}

}  // extern "C"
