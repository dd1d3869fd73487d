// neon_longctx.cuh -- helpers shared by the long-context operators' kernels
// (neon_rope.cu, neon_kv8.cu): typed loads and stores, programmatic dependent
// launch, mbarriers and bulk copies, and the host-side argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cmath>
#include <string>

#include "neon_cuda.h"
#include "neon_internal.h"

namespace longctx {

constexpr unsigned kErrWait = 1u;  // device error word: a bounded wait ran out

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---- values of the three element types ----

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Four values of T in one load.
template <typename T>
struct alignas(4 * sizeof(T)) Vec4 {
    T t[4];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (sizeof(T) == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            *reinterpret_cast<uint4*>(t) = v;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            *reinterpret_cast<uint2*>(t) = v;
        }
    }
};

// fp32 pairs in one instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// ---- mbarriers and bulk copies (one warp or CTA of its own shared memory) ----

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
// dst, src and bytes are multiples of 16
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_addr(dst)),
                 "l"(src), "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return done != 0;
}
// Whether a phase has completed, without waiting.
__device__ __forceinline__ bool bar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return done != 0;
}
// Waits for a phase; gives up after about 2 s, notes it in *err and returns false.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, unsigned* err) {
    if (bar_try(bar, parity)) return true;
    uint64_t t0, t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    for (;;) {
        if (bar_try(bar, parity)) return true;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
        if (t - t0 > 2000000000ull) {
            atomicOr(err, kErrWait);
            return false;
        }
    }
}

// ---- host ----

inline size_t type_bytes(int type) { return type == NEON_GGML_F32 ? 4 : type == NEON_GGML_F16 || type == NEON_GGML_BF16 ? 2 : 0; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Whether n rows of x and n of y, each its stride and length in bytes, have no byte in common: rows of one buffer
// side by side have not.
inline bool apart(const void* px, size_t xs, size_t xrow, const void* py, size_t ys, size_t yrow, size_t n) {
    const char *x = (const char*)px, *y = (const char*)py;
    if (x + (n - 1) * xs + xrow <= y || y + (n - 1) * ys + yrow <= x) return true;
    if (xs != ys || n == 1) return false;
    const size_t d = x < y ? (size_t)(y - x) % xs : (xs - (size_t)(x - y) % xs) % xs;  // y's place in a row of x
    return d >= xrow && d + yrow <= xs;
}

// A buffer that a call reads or writes.
struct Range {
    const void* p;
    size_t bytes;
    bool meets(const Range& o) const {
        return bytes && o.bytes && (const char*)p < (const char*)o.p + o.bytes && (const char*)o.p < (const char*)p + bytes;
    }
};

// Runs a scope with the device of a buffer current.
struct OnDevice {
    int prev = -1, device = -1, rc = NEON_OK;
    explicit OnDevice(const void* p) {
        cudaPointerAttributes a{};
        cudaError_t e = cudaPointerGetAttributes(&a, p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            rc = neon_internal::cuda_error(e, "cudaPointerGetAttributes");
            return;
        }
        if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) {
            rc = neon_internal::error(NEON_ERR_INVALID, "not a device buffer");
            return;
        }
        device = a.device;
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != device && (e = cudaSetDevice(device)) != cudaSuccess) rc = neon_internal::cuda_error(e, "cudaSetDevice");
    }
    ~OnDevice() {
        if (prev >= 0 && prev != device && device >= 0) cudaSetDevice(prev);
    }
};

template <typename... KArgs, typename... Args>
int launch(const char* what, void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster,
           Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (neon_internal::pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)cluster;
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
    if (e != cudaSuccess) return neon_internal::cuda_error(e, what);
    return neon_internal::launched(1);
}

// The frequencies of a checked rotation, in turns per position (f_i / 2 pi).
struct RopeTurns {
    double f[128];
};
int rope_check(const neon_rope_t* r, size_t head_dim);
int rope_turns(const neon_rope_t& r, RopeTurns* t);

// cos and sin of 2 pi * turns * pos: the whole turns drop out in 64 bits (an
// int32 position times a turn has an error of 2^-53 of its size), the rest is
// at most half a turn and goes through fp32.
__device__ __forceinline__ float2 turn(double turns, int pos) {
    const double a = turns * (double)pos;
    const float r = 2.f * (float)(a - rint(a));
    float s, c;
    sincospif(r, &s, &c);
    return make_float2(c, s);
}

}  // namespace longctx
