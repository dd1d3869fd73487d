// neon_kv8.h -- the 8-bit KV cache's launchers, shared by its entry points and
// the decode engine (arguments already checked, the device current).
#pragma once

#include <cuda_runtime.h>

#include "neon_cuda.h"

namespace longctx {

int kv8_check(const neon_kv8_t* c);          // shape
int kv8_check_buffers(const neon_kv8_t* c);  // shape and pointers
int kv8_append(const neon_kv8_t& c, const void* k, size_t ks, const void* v, size_t vs, size_t n, int type, int device,
               cudaStream_t st);
// (a caller that never asks for weights needs no room for the stored scores and queries that they are made from)
size_t kv8_attention_workspace(const neon_kv8_t& c, size_t n, size_t n_head, bool weights);
int kv8_attention(const neon_kv8_t& c, const void* q, size_t qs, void* o, size_t os, size_t n, size_t n_head,
                  float scale, int type, float* weight, void* ws, int device, cudaStream_t st);
int kv8_evict(const neon_kv8_t& src, const float* w, const neon_kv8_t& dst, float* wd, size_t keep, size_t sink,
              size_t recent, const neon_rope_t* rope, int32_t* kept, cudaStream_t st);
// The rows kept[n_kv_head][keep] (ascending, -1 behind the last) of src into dst; weights too unless null.
int kv8_move(const neon_kv8_t& src, const float* w, const neon_kv8_t& dst, float* wd, size_t keep, const neon_rope_t* rope,
             const int32_t* kept, cudaStream_t st);
// Rows [row0, row1) as zeros without weight (w unless null), like rows of a new cache; those before them keep their
// values and their tail, what lies behind them in the last block goes too.
int kv8_clear(const neon_kv8_t& c, float* w, size_t row0, size_t row1, cudaStream_t st);

}  // namespace longctx
