// 4-bit key/value cache: argument checks, the batch's token bookkeeping and
// the nibble unpacking shared by its kernels.
//
// Formats (include/openquant_b200.h): codes [pages][kv_heads][page_size]
// [head_dim / 2] bytes, scales fp16 [...][head_dim / group].  A scale has 8
// significant bits and a code 3, so code * scale is exact in fp16: the
// tensor-core kernels multiply the cached values without rounding them.
#pragma once

#include "oq_sm100.cuh"

namespace oq {
namespace kv4 {

constexpr int kMaxSequences = 2048;
constexpr float kMaxScale = 9344.0f;  // 146 * 64 (8 bits), 7 * 9344 = 65408 <= fp16's 65504
constexpr int OQ_DEV_INDEX = 3;

// Error word of the cache kernels (a page or position outside its arrays).
// Unlike the pipelined kernels' word it stops nothing.
static __device__ int g_index_error;

__device__ __forceinline__ void index_error() { atomicCAS(&g_index_error, 0, OQ_DEV_INDEX); }

static int take_index_error(int *code) {
    int v = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_index_error, sizeof(int)) != cudaSuccess) return OQ_ERR_CUDA;
    if (v != 0 && cudaMemcpyToSymbol(g_index_error, &zero, sizeof(int)) != cudaSuccess) return OQ_ERR_CUDA;
    if (v != 0 && *code == 0) *code = v;
    return OQ_OK;
}

namespace {
struct IndexErrorRegistration {
    IndexErrorRegistration() { register_device_error_reader(&take_index_error); }
};
static IndexErrorRegistration g_index_error_registration;
}  // namespace

struct Batch {
    const int32_t *table, *lengths, *starts;
    int sequences, max_pages;
};

// First token and token count of sequence b, kept inside the step's array.
// False: its starts are not in order within the array (the first one at 0).
__device__ __forceinline__ bool tokens_of(const Batch &bt, int b, int64_t tokens, int &first, int &count) {
    if (bt.starts == nullptr) {
        first = b;
        count = b < tokens ? 1 : 0;
        return true;
    }
    const int s = __ldg(bt.starts + b), e = __ldg(bt.starts + b + 1);
    first = b == 0 ? 0 : min(max(s, 0), (int)tokens);
    count = min(max(e, first), (int)tokens) - first;
    return s == first && e == first + count;
}

// Cached tokens of sequence b that its page-table row has room for; `end`: its
// length as it is, from which the step's tokens have their positions.
__device__ __forceinline__ int length_of(const Batch &bt, int b, int page_size, int &end) {
    const int64_t cap = (int64_t)bt.max_pages * page_size;
    const int n = __ldg(bt.lengths + b);
    end = max(n, 0);
    if (n < 0 || n > cap) {
        index_error();
        return n < 0 ? 0 : (int)cap;
    }
    return n;
}

// Sequence of token t (all 32 lanes take part, t uniform): the number of
// starts[1..] that are <= t.  bt.sequences or more for a padding token.
__device__ __forceinline__ int sequence_of(const Batch &bt, int t) {
    if (bt.starts == nullptr) return t;
    const int lane = threadIdx.x & 31;
    int seq = 0;
    for (int base = 0; base < bt.sequences; base += 32) {
        const int i = base + lane;
        const bool in = i < bt.sequences && __ldg(bt.starts + i + 1) <= t;
        const int c = __popc(__ballot_sync(0xffffffffu, in));
        seq += c;
        if (c < 32) break;
    }
    return seq;
}

// The eight codes of a word as fp16 integers.  The word holds codes n0..n7 (two's
// complement); r[j] = {n_j, n_(j+4)} as exact fp16 integers: one LOP3 puts
// u = n + 8 into the mantissa of 1024 (low nibble class) or 16 u into it
// (next class), and one add or FMA takes the offset away exactly.
__device__ __forceinline__ uint32_t lop_and_xor(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2 *>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t *>(&v); }

__device__ __forceinline__ void unpack_int(uint32_t w, __half2 (&r)[4]) {
    const __half2 off = __half2half2(__ushort_as_half(0x6408));   // 1032
    const __half2 six = __half2half2(__ushort_as_half(0x2C00));   // 1 / 16
    const __half2 off2 = __half2half2(__ushort_as_half(0xD480));  // -72
    const uint32_t h = w >> 8;
    r[0] = __hsub2(as_half2(lop_and_xor(w, 0x000F000Fu, 0x64086408u)), off);
    r[1] = __hfma2(as_half2(lop_and_xor(w, 0x00F000F0u, 0x64806480u)), six, off2);
    r[2] = __hsub2(as_half2(lop_and_xor(h, 0x000F000Fu, 0x64086408u)), off);
    r[3] = __hfma2(as_half2(lop_and_xor(h, 0x00F000F0u, 0x64806480u)), six, off2);
}

// Host: checks a cache and a batch (OQ_ERR_INVALID with a message).
int check_cache(const oq_kv4_cache *c);
int check_batch(const oq_kv4_batch *b, int64_t tokens);

inline Batch device_batch(const oq_kv4_batch *b) {
    return Batch{b->page_table, b->lengths, b->starts, b->sequences, b->max_pages};
}

}  // namespace kv4
}  // namespace oq
