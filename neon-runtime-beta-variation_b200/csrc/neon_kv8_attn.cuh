// neon_kv8_attn.cuh -- what the kernels of the attention over the 8-bit KV
// cache share (neon_kv8_attn.cu: few query rows, joins, weights;
// neon_kv8_prompt.cu: many query rows on tcgen05).
#pragma once

#include "neon_longctx.cuh"
#include "neon_kv8.h"

namespace longctx {

// ---- codes and fp32 values as fp16 ----

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// 1024 + u is the half 0x6400 | u for a byte u; with u = code + 128 the code is
// that less 1152, exactly.
__device__ __forceinline__ uint32_t unbias(uint32_t h) { return h2_bits(__hsub2(bits_h2(h), bits_h2(0x64806480u))); }
// bytes 0, 1 and 2, 3 of a word of codes + 128 as two half2
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) { return unbias(__byte_perm(w, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) { return unbias(__byte_perm(w, 0x64646464u, 0x4342)); }

// x, y as hi and lo half2 terms
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(x - f.x, y - f.y));
}

__device__ __forceinline__ float q_value(const void* q, int type, long long i) {
    return type == NEON_GGML_F32   ? ((const float*)q)[i]
           : type == NEON_GGML_F16 ? __half2float(((const __half*)q)[i])
                                   : __bfloat162float(((const __nv_bfloat16*)q)[i]);
}
__device__ __forceinline__ void o_store(void* o, int type, long long i, float v) {
    if (type == NEON_GGML_F32) ((float*)o)[i] = v;
    else if (type == NEON_GGML_F16) ((__half*)o)[i] = __float2half_rn(v);
    else ((__nv_bfloat16*)o)[i] = __float2bfloat16_rn(v);
}

// 2^x; below 2^-126: 0
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 .. 127

// The rows that token t may attend to.
__device__ __forceinline__ int keys_of(int past, int t, int cap) {
    return (int)max(0LL, min((long long)past + t + 1, (long long)cap));
}

// Rows of one KV head: row r is query head r % group of token r / group.
struct AttnArgs {
    neon_kv8_t c;
    const void* q;
    void* o;
    long long qs, os;
    int n, n_head, group, type;
    float scale;     // softmax scale * log2(e)
    float* weight;
    int nsplit;      // shares of a unit's keys at most
    int unit;        // rows of a CTA of the main kernel (8, 16 or a prompt unit)
    int min_tiles;   // tiles before another CTA joins
    int tile_shift;  // log2 of a tile's keys
    float* stats;    // [H][rows][2]: a row's final m and 1 / l (0 for a row without keys)
    float* part_o;   // [H][rows][nsplit][hd]: o of a split, not normalised, in units of
    float* part_ml;  // [H][rows][nsplit][2]: 2^m with m, and l
    float* scores;   // few rows, weights kept: [H][rows, to whole units][capacity] scores * log2(e), or null
    float4* sums;    // prompts: o of the chains of a row that are done, see put_by
    // prompts: query tiles of 128 rows as fp16 (put_queries in neon_kv8_prompt.cu), and the rows' factors
    unsigned char* qt;
    float* qfactor;
    unsigned* err;
};

// How the keys of a unit of rows are shared out: `per` tiles a CTA, as many CTAs as that takes (split * per < tiles;
// one at least). Few divisions: they are a good part of a short call.
struct Shares {
    int tiles, per;
    __device__ __forceinline__ bool whole() const { return per >= tiles; }
    __device__ __forceinline__ bool has(int split) const { return split == 0 || split * per < tiles; }
    __device__ __forceinline__ int count() const { return whole() ? 1 : (tiles + per - 1) / per; }
};
__device__ __forceinline__ int token_of(const AttnArgs& a, int row) { return a.n == 1 ? 0 : row / a.group; }
__device__ __forceinline__ Shares shares_of(const AttnArgs& a, int past, int unit) {
    const int rows = a.n * a.group;
    const int last = token_of(a, min(unit * a.unit + a.unit - 1, rows - 1));
    Shares s;
    s.tiles = (keys_of(past, last, (int)a.c.capacity) + (1 << a.tile_shift) - 1) >> a.tile_shift;
    s.per = a.nsplit == 1 ? s.tiles : max((s.tiles + a.nsplit - 1) / a.nsplit, min(s.tiles, a.min_tiles));
    return s;
}

// Query rows of a KV head above which the prompt kernel takes them. Over 20000 rows of 8 heads x 128 the rows kernel
// takes 32 rows in 41 us (fp32) and 32 us (bf16), the prompt kernel in 59 and 47; over 120000 it is 181 and 112
// against 250 and 199. At 64 rows the prompt kernel is ahead for fp32 (59 against 71 us over 20000).
constexpr int kPromptRows = 32;

// Keys whose outputs a prompt's products sum in one go, in fp32 and in types of 16 bits; longer shares are added up in
// fp32 in the workspace (kv8_prompt_kernel's put_by). The products cut their sums off instead of rounding them, so what
// came early in a sum fades: one sum over n keys leaves an output 1.4e-9 n off. 600 tokens of 64 / 8 heads x 128 in
// fp32, error against float64 and time: over 4600 rows 1.1e-6 and 282 us (one sum: 5.0e-6 and 253; sums of 2048 keys:
// 2.2e-6 and 263; an fp32 product's 1.3e-6), over 16600 rows 1.1e-6 and 1080 us (one sum: 2.1e-5 and 920), over 120600
// 1.3e-6 and 8.6 ms (1.6e-4 and 7.7). 4096 keys' 5.7e-6 is a fortieth of an fp16 output's rounding.
constexpr int kChainKeys = 1024, kChainKeys16 = 4096;

constexpr float kLog2e = 1.4426950408889634f;

// Prompts (neon_kv8_prompt.cu): bytes of the query tiles, and the launches.
size_t prompt_query_bytes(const neon_kv8_t& c, size_t rows, int type);
int prompt_unit(int hd);
int prompt_tile_shift();
int launch_prompt(const AttnArgs& a, cudaStream_t st);
int launch_prompt_weights(const AttnArgs& a, cudaStream_t st);  // after launch_prompt and its joins

}  // namespace longctx
