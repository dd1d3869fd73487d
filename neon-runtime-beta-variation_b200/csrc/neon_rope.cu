// neon_rope.cu -- rotary positions (neon_cuda_rope).
//
//   y_a = m (x_a cos t - x_b sin t),  y_b = m (x_a sin t + x_b cos t),  t = pos f_i
//
// for the pairs (a, b) of each head's first n_dims values; the rest is copied.
// Each value is read and written once, so memory bounds it. A CTA takes some
// heads of some positions: it first puts the positions' cos and sin into
// shared memory (once for all heads; the 64-bit reduction of the angle is the
// costly part), then streams the heads in 16-byte pieces.
#include "neon_longctx.cuh"

#include <algorithm>

namespace longctx {

int rope_check(const neon_rope_t* r, size_t head_dim) {
    using neon_internal::error;
    if (!r) return error(NEON_ERR_INVALID, "null rope");
    if (r->n_dims < 2 || r->n_dims % 2 || r->n_dims > 256 || r->n_dims > head_dim)
        return error(NEON_ERR_INVALID, "rope: n_dims must be even, from 2 to 256 and at most head_dim");
    if (r->layout != NEON_ROPE_INTERLEAVED && r->layout != NEON_ROPE_HALF)
        return error(NEON_ERR_INVALID, "rope: unknown layout");
    if (!(r->base > 0) || !std::isfinite(r->base) || !(r->scale > 0) || !std::isfinite(r->scale))
        return error(NEON_ERR_INVALID, "rope: base and scale must be positive");
    if (!std::isfinite((float)r->magnitude)) return error(NEON_ERR_INVALID, "rope: magnitude must be finite in fp32");
    if (!(r->yarn >= 0 && r->yarn <= 1)) return error(NEON_ERR_INVALID, "rope: yarn must be from 0 to 1");
    if (r->yarn > 0 && (r->orig_ctx == 0 || !(r->beta_slow > 0) || !(r->beta_fast >= r->beta_slow) ||
                        !std::isfinite(r->beta_fast) || r->base == 1.0))
        return error(NEON_ERR_INVALID, "rope: yarn needs orig_ctx, beta_fast >= beta_slow > 0 and a base other than 1");
    if (r->factors)
        for (uint32_t i = 0; i < r->n_dims / 2; ++i)
            if (!(r->factors[i] > 0) || !std::isfinite(r->factors[i]))
                return error(NEON_ERR_INVALID, "rope: factors must be positive");
    return NEON_OK;
}

int rope_turns(const neon_rope_t& r, RopeTurns* t) {
    const double pi2 = 6.283185307179586476925286766559;
    const double den = r.freq_dim ? r.freq_dim : r.n_dims;
    double lo = 0, hi = 0;
    if (r.yarn > 0) {
        auto at = [&](double beta) { return r.n_dims * std::log(r.orig_ctx / (pi2 * beta)) / (2 * std::log(r.base)); };
        lo = std::max(0.0, std::floor(at(r.beta_fast)));
        hi = std::min((double)r.n_dims - 1, std::ceil(at(r.beta_slow)));
    }
    // the powers by products in 80 bits (64 of them lose 2^-58): a pow for each would be half of a short call
    const long double step = powl((long double)r.base, -2.0L / den);
    long double power = 1;
    for (uint32_t i = 0; i < 128; ++i, power *= step) {
        t->f[i] = 0;
        if (i >= r.n_dims / 2) continue;
        double f = (double)power;
        if (r.factors) f /= r.factors[i];
        double own = 0;
        if (r.yarn > 0)
            own = r.yarn * (1 - std::min(1.0, std::max(0.0, ((double)i - lo) / std::max(hi - lo, 0.001))));
        t->f[i] = (f / r.scale * (1 - own) + f * own) / pi2;
        if (!std::isfinite(t->f[i])) return neon_internal::error(NEON_ERR_INVALID, "rope: a frequency beyond the range of doubles");
    }
    return NEON_OK;
}

namespace {

constexpr int kMaxTargets = 4;
constexpr int kThreads = 256;
constexpr int kMaxTile = 16;  // positions per CTA at most: a table of 16 x 128 (cos, sin) is 16 KB

struct RopeArgs {
    const void* x[kMaxTargets];
    void* y[kMaxTargets];
    long long xs[kMaxTargets], ys[kMaxTargets];
    int head0[kMaxTargets + 1];  // the targets' heads, counted through
    const int* pos;
    int n, hd, pairs;   // pairs = n_dims / 2
    int tile, heads;    // positions and heads of a CTA
    int back;
    float mag;
    RopeTurns turns;
};

// One piece of a head: V values for the interleaved layout; for the halves
// layout V values of the first half with their partners, and after those the
// V-value pieces that are copied.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(kThreads, 4) rope_kernel(const __grid_constant__ RopeArgs a) {
    extern __shared__ float2 cs[];
    pdl_wait();
    pdl_trigger();
    const int t0 = blockIdx.x * a.tile, h0 = blockIdx.y * a.heads;
    const int nt = min(a.tile, a.n - t0), nh = min(a.heads, a.head0[kMaxTargets] - h0);
    const int per = HALF ? (a.hd - a.pairs) / V : a.hd / V;  // pieces of a head
    const int total = nt * nh * per;
    for (int i = threadIdx.x; i < nt * a.pairs; i += kThreads) {
        const int t = i / a.pairs, p = i - t * a.pairs;
        float2 c = turn(a.turns.f[p], a.pos[t0 + t]);
        if (a.back) c.y = -c.y;
        cs[i] = make_float2(c.x * a.mag, c.y * a.mag);
    }
    __syncthreads();

    int v = threadIdx.x % per, h = threadIdx.x / per, t = h / nh;
    h -= t * nh;
    const int dv = kThreads % per, dh = kThreads / per;
    constexpr int U = 2;
    for (int i = threadIdx.x; i < total; i += U * kThreads) {
        alignas(16) T lo[U][V], hi[U][V];
        T *dst[U];
        int vv[U], tt[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool on = i + u * kThreads < total;
            vv[u] = on ? v : -1;
            tt[u] = t;
            if (on) {
                const int hh = h0 + h;
                int g = 0;
#pragma unroll
                for (int k = 1; k < kMaxTargets; ++k) g += hh >= a.head0[k];
                const long long col = (long long)(hh - a.head0[g]) * a.hd;
                const T* src = (const T*)a.x[g] + (t0 + t) * a.xs[g] + col;
                dst[u] = (T*)a.y[g] + (t0 + t) * a.ys[g] + col;
                const bool rot = !HALF || v * V < a.pairs;
                const int e = rot ? v * V : v * V + a.pairs;  // first value of the piece
                if constexpr (V * sizeof(T) == 16) {
                    *reinterpret_cast<uint4*>(lo[u]) = *reinterpret_cast<const uint4*>(src + e);
                    if (HALF && rot) *reinterpret_cast<uint4*>(hi[u]) = *reinterpret_cast<const uint4*>(src + e + a.pairs);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) lo[u][j] = src[e + j];
                    if (HALF && rot)
#pragma unroll
                        for (int j = 0; j < V; ++j) hi[u][j] = src[e + a.pairs + j];
                }
            }
            v += dv;
            h += dh;
            if (v >= per) { v -= per; ++h; }
            while (h >= nh) { h -= nh; ++t; }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (vv[u] < 0) continue;
            const bool rot = HALF ? vv[u] * V < a.pairs : vv[u] * V < 2 * a.pairs;
            const int e = HALF && !rot ? vv[u] * V + a.pairs : vv[u] * V;
            if (rot) {
                const float2* c = cs + tt[u] * a.pairs;
                if (HALF) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float2 w = c[e + j];
                        const float p = to_f(lo[u][j]), q = to_f(hi[u][j]);
                        lo[u][j] = from_f<T>(__fmaf_rn(p, w.x, -__fmul_rn(q, w.y)));
                        hi[u][j] = from_f<T>(__fmaf_rn(p, w.y, __fmul_rn(q, w.x)));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j + 1 < V; j += 2) {
                        const float2 w = c[(e + j) / 2];
                        const float p = to_f(lo[u][j]), q = to_f(lo[u][j + 1]);
                        lo[u][j] = from_f<T>(__fmaf_rn(p, w.x, -__fmul_rn(q, w.y)));
                        lo[u][j + 1] = from_f<T>(__fmaf_rn(p, w.y, __fmul_rn(q, w.x)));
                    }
                }
            }
            if constexpr (V * sizeof(T) == 16) {
                *reinterpret_cast<uint4*>(dst[u] + e) = *reinterpret_cast<const uint4*>(lo[u]);
                if (HALF && rot) *reinterpret_cast<uint4*>(dst[u] + e + a.pairs) = *reinterpret_cast<const uint4*>(hi[u]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) dst[u][e + j] = lo[u][j];
                if (HALF && rot)
#pragma unroll
                    for (int j = 0; j < V; ++j) dst[u][e + a.pairs + j] = hi[u][j];
            }
        }
    }
}

using RopeKernel = void (*)(RopeArgs);
template <typename T>
RopeKernel rope_kernel_for(bool vec, bool half) {
    constexpr int V = 16 / (int)sizeof(T);
    // single pieces: one pair (interleaved) or one value with its partner (halves)
    if (vec) return half ? rope_kernel<T, V, true> : rope_kernel<T, V, false>;
    return half ? rope_kernel<T, 1, true> : rope_kernel<T, 2, false>;
}

}  // namespace
}  // namespace longctx

using namespace longctx;
using neon_internal::error;

extern "C" int neon_cuda_rope(const neon_rope_t* rope, int type, const int32_t* d_pos, size_t n, size_t head_dim,
                              const neon_rope_target_t* targets, size_t n_targets, int backward, void* stream) {
    int rc = rope_check(rope, head_dim);
    if (rc) return rc;
    const size_t eb = type_bytes(type);
    if (!eb) return error(NEON_ERR_UNSUPPORTED, "rope: type must be F32, F16 or BF16");
    if (head_dim % 2 || head_dim > 1024) return error(NEON_ERR_INVALID, "rope: head_dim must be even and at most 1024");
    if (!targets || n_targets == 0 || n_targets > (size_t)kMaxTargets)
        return error(NEON_ERR_INVALID, "rope: 1 to 4 targets");
    if (n == 0) return NEON_OK;
    if (!d_pos || !aligned(d_pos, 4)) return error(NEON_ERR_INVALID, "rope: null or unaligned positions");
    if (n > (size_t)INT32_MAX / 2) return error(NEON_ERR_INVALID, "rope: too many positions");
    RopeArgs a{};
    const bool half = rope->layout == NEON_ROPE_HALF;
    const size_t V = 16 / eb;
    bool vec = head_dim % V == 0 && (half ? rope->n_dims / 2 : rope->n_dims) % V == 0;
    size_t heads = 0;
    for (size_t g = 0; g < (size_t)kMaxTargets; ++g) {
        a.head0[g] = (int)heads;
        if (g >= n_targets) continue;
        const neon_rope_target_t& t = targets[g];
        const size_t row = t.n_heads * head_dim;
        if (!t.X || !t.Y) return error(NEON_ERR_INVALID, "rope: null buffer");
        if (t.n_heads == 0 || t.n_heads > 65535) return error(NEON_ERR_INVALID, "rope: a target needs 1 to 65535 heads");
        if (t.x_stride < row || t.y_stride < row) return error(NEON_ERR_INVALID, "rope: stride smaller than the heads");
        if (!aligned(t.X, eb) || !aligned(t.Y, eb)) return error(NEON_ERR_INVALID, "rope: buffer not aligned to its type");
        if (t.X == t.Y) {
            if (t.x_stride != t.y_stride && n > 1) return error(NEON_ERR_INVALID, "rope: in place, the strides must be equal");
        } else if (!apart(t.X, t.x_stride * eb, row * eb, t.Y, t.y_stride * eb, row * eb, n)) {
            return error(NEON_ERR_INVALID, "rope: X and Y overlap");
        }
        for (size_t k = 0; k < g; ++k) {
            const neon_rope_target_t& u = targets[k];
            const size_t other = u.n_heads * head_dim * eb;
            if (!apart(t.Y, t.y_stride * eb, row * eb, u.Y, u.y_stride * eb, other, n) ||
                !apart(t.Y, t.y_stride * eb, row * eb, u.X, u.x_stride * eb, other, n) ||
                !apart(t.X, t.x_stride * eb, row * eb, u.Y, u.y_stride * eb, other, n))
                return error(NEON_ERR_INVALID, "rope: a target's Y overlaps another target");
        }
        vec = vec && aligned(t.X, 16) && aligned(t.Y, 16) && (n == 1 || (t.x_stride % V == 0 && t.y_stride % V == 0));
        a.x[g] = t.X;
        a.y[g] = t.Y;
        a.xs[g] = (long long)t.x_stride;
        a.ys[g] = (long long)t.y_stride;
        heads += t.n_heads;
    }
    a.head0[kMaxTargets] = (int)heads;
    for (size_t g = n_targets; g < (size_t)kMaxTargets; ++g) a.head0[g] = (int)heads;
    rc = rope_turns(*rope, &a.turns);
    if (rc) return rc;
    OnDevice dev(targets[0].Y);
    if (dev.rc) return dev.rc;
    const int sms = neon_internal::device_sms(dev.device);
    if (sms < 0) return NEON_ERR_CUDA;
    a.pos = d_pos;
    a.n = (int)n;
    a.hd = (int)head_dim;
    a.pairs = (int)rope->n_dims / 2;
    a.back = backward != 0;
    a.mag = (float)rope->magnitude;
    // Pieces per CTA: one to four a thread, so that CTAs in their table and CTAs in their heads share the SMs (4099
    // positions of 32 heads: 16 us; always one 28, always four 16; one position of 24 heads: 2.2, always four 2.7).
    const int V1 = vec ? (int)V : half ? 1 : 2;
    const long long per = half ? (a.hd - a.pairs) / V1 : a.hd / V1, row = per * (long long)heads;
    const long long want = std::min<long long>(std::max<long long>((long long)n * row / (sms * 4), kThreads), 4 * kThreads);
    a.tile = (int)std::min<long long>({std::max<long long>(1, want / row), (long long)kMaxTile, (long long)n});
    a.heads = row <= want ? (int)heads : (int)std::max<long long>(std::min<long long>(want / per, (long long)heads), 1);
    a.heads = std::max(a.heads, (int)((heads + 65534) / 65535));  // (grid.y is at most 65535)
    const dim3 grid((unsigned)((n + a.tile - 1) / a.tile), (unsigned)((heads + a.heads - 1) / a.heads));
    RopeKernel k = type == NEON_GGML_F32   ? rope_kernel_for<float>(vec, half)
                   : type == NEON_GGML_F16 ? rope_kernel_for<__half>(vec, half)
                                           : rope_kernel_for<__nv_bfloat16>(vec, half);
    return launch("rope_kernel", k, grid, kThreads, (size_t)a.tile * a.pairs * sizeof(float2), (cudaStream_t)stream, 1, a);
}
