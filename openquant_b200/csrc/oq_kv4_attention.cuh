// Arguments shared by the attention kernels of the 4-bit key/value cache.
#pragma once

#include "oq_kv4.cuh"

namespace oq {
namespace kv4 {

constexpr float kLift = 6.0f;    // a running maximum is set this much below the largest score (log2)
constexpr float kRaise = 14.0f;  // and raised when a score passes it by more than this

// Scores beyond this (log2) are rounded to fp32 before the maximum is taken off.
// One fused operation would take the exact product s f less a maximum that was
// rounded: up to |s f| 2^-23 too much, and from 2^24 on p may pass fp16.
// (Beyond 2^26 fp32 numbers lie further apart than kLift: the largest p of a
// row is then 1 to 2^8.)
constexpr float kHuge = 1048576.0f;

constexpr float kNone = -3e38f;  // the maximum of no scores: finite, below what a score can be

struct AttnArgs {
    const uint8_t *k_codes, *v_codes;
    const __half *k_scales, *v_scales;
    int64_t pages;
    int page_size, kv_heads;
    Batch batch;
    const void *q;
    int64_t q_ts, q_hs;
    void *out;
    float *log_sum;
    int64_t tokens;
    int q_heads, ratio;  // ratio: query heads a key head
    float f;             // scale * log2 e
    int64_t window;
    int causal;
    float *parts;    // partial results
    int vec;         // q rows 16-byte aligned
    int max_tokens;  // what the launches are planned for: a sequence with more tokens is left out
    int few;         // sequences of at most `few` query rows a key head go to the streaming kernel,
                     // the others to the prompt kernel
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ void put(T *p, float v);
template <> __device__ __forceinline__ void put<__half>(__half *p, float v) { *p = __float2half_rn(v); }
template <> __device__ __forceinline__ void put<__nv_bfloat16>(__nv_bfloat16 *p, float v) {
    *p = __float2bfloat16_rn(v);
}

// Eight query elements as fp32; vec: 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load_q8(const T *p, bool vec, float (&v)[8]) {
    alignas(16) T e[8];
    if (vec) {
        *reinterpret_cast<uint4 *>(e) = __ldg(reinterpret_cast<const uint4 *>(p));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Elem<T>::to_f32(e[i]);
}

// Queries in bf16 go to fp16 times a power of two per row that brings the
// largest element to [2^8, 2^9): exact but for elements 2^-22 below it (whose
// low bits fall under fp16's smallest step).  Returns that power; scores are
// multiplied by its inverse (`down`).  fp16 queries are taken as they are.
template <typename T>
__device__ __forceinline__ float fp16_power(float top, float &down) {
    down = 1.0f;
    if (std::is_same<T, __half>::value) return 1.0f;
    const int ex = (int)(__float_as_uint(top) >> 23);  // biased; 0: zero or subnormal, 255: inf
    if (ex == 0 || ex == 255) return 1.0f;
    const int sh = min(135 - ex, 100);
    down = __uint_as_float((uint32_t)(127 - sh) << 23);
    return __uint_as_float((uint32_t)(127 + sh) << 23);
}

// The prompt kernel over every sequence with more than a.few query rows.
// `items`: an upper bound of its (sequence, key head, row block) items, each
// of which is cut into up to `cuts` parts of its cached tokens.
constexpr int kPromptRows = 256;  // query rows of an item
constexpr int kMostCuts = 64;
int prompt_cuts(const oq_kv4_cache *c, const oq_kv4_batch *b, int64_t items);
int64_t prompt_part_bytes(const oq_kv4_cache *c, int64_t items, int cuts);
int prompt_attention(const AttnArgs &a, int dtype, const oq_kv4_cache *c, int64_t items, int cuts, cudaStream_t st);

}  // namespace kv4
}  // namespace oq
