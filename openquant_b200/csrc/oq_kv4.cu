// Rotary positions, append to and read from the 4-bit key/value cache.
#include "oq_kv4.cuh"

namespace oq {
namespace kv4 {

int check_cache(const oq_kv4_cache *c) {
    OQ_REQUIRE(c != nullptr, "null cache");
    OQ_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128");
    OQ_REQUIRE(c->group_size == 32 || c->group_size == 64 || c->group_size == 128,
               "Group size must be 32, 64 or 128");
    OQ_REQUIRE(c->group_size <= c->head_dim, "Group size must be at most head_dim");
    OQ_REQUIRE(c->page_size >= 16 && c->page_size % 16 == 0, "page_size must be a positive multiple of 16");
    OQ_REQUIRE(c->pages >= 1 && c->kv_heads >= 1, "Cache dimensions must be positive");
    // 16-row blocks are counted in 32 bits
    OQ_REQUIRE(c->pages <= (1ll << 31) - 1 && c->pages * c->kv_heads <= (1ll << 31) / (c->page_size / 16),
               "cache too large");
    OQ_REQUIRE(c->k_codes && c->k_scales && c->v_codes && c->v_scales, "null pointer argument");
    OQ_REQUIRE(aligned(c->k_codes, 16) && aligned(c->k_scales, 16) && aligned(c->v_codes, 16) &&
                   aligned(c->v_scales, 16),
               "cache arrays must be 16-byte aligned");
    return OQ_OK;
}

int check_batch(const oq_kv4_batch *b, int64_t tokens) {
    OQ_REQUIRE(b != nullptr, "null batch");
    OQ_REQUIRE(b->sequences >= 1 && b->sequences <= kMaxSequences, "a batch has 1 to %d sequences", kMaxSequences);
    OQ_REQUIRE(b->max_pages >= 1, "the page table needs at least one page per sequence");
    OQ_REQUIRE(b->page_table && b->lengths, "null pointer argument");
    OQ_REQUIRE(b->max_tokens >= 1, "max_tokens must be positive");
    OQ_REQUIRE(tokens >= 1 && tokens < (1ll << 31), "the token count must be positive and below 2^31");
    OQ_REQUIRE(b->starts != nullptr || b->max_tokens == 1, "max_tokens > 1 needs starts");
    return OQ_OK;
}

namespace {

constexpr int kWarps = 4;  // warps per CTA
constexpr int kRows = 4;   // head rows of a lane in one step (and as many in flight)

struct Rotary {
    const float *table;
    int64_t rows;
    int dim, flags;
    const void *positions;
    int wide;
    float one = 1.0f;  // see turn2()
};

struct Rows {  // [tokens][heads][head_dim] with strides in elements
    const void *p;
    int64_t ts, hs;
};

// How a lane finds the partners of its eight elements.
enum Pairs {
    kNone,     // no rotation
    kShuffle,  // half layout, dim / 2 a multiple of 8: eight elements of one other lane
    kNext,     // interleaved, dim a multiple of 8: the lane's own neighbours
    kAny,      // any other dim: half-layout partners from memory
};

int pairs_of(const Rotary &r) {
    if (r.table == nullptr) return kNone;
    if (r.flags & OQ_ROTARY_INTERLEAVED) return r.dim % 8 == 0 ? kNext : kAny;
    return r.dim % 16 == 0 ? kShuffle : kAny;
}

__device__ __forceinline__ int64_t position_at(const Rotary &r, int64_t t) {
    return r.wide ? __ldg(static_cast<const long long *>(r.positions) + t)
                  : (int64_t)__ldg(static_cast<const int *>(r.positions) + t);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// Eight consecutive elements as they are in memory.
template <typename T>
struct alignas(16) Eight {
    T e[8];
};

// VEC: 16-byte aligned.  Plain loads (not the read-only path): the output may
// be the input.
template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T *p, Eight<T> &v) {
    if (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            reinterpret_cast<uint4 *>(v.e)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.e[i] = p[i];
    }
}

template <typename T>
__device__ __forceinline__ void widen(const Eight<T> &v, float2 (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = make_float2(Elem<T>::to_f32(v.e[2 * i]), Elem<T>::to_f32(v.e[2 * i + 1]));
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_row8(T *p, const float2 (&v)[4]) {
    alignas(16) T e[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        e[2 * i] = from_f32<T>(v[i].x);
        e[2 * i + 1] = from_f32<T>(v[i].y);
    }
    if (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(e)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = e[i];
    }
}

// A lane's eight elements [8c, 8c + 8) of a head: the cos and signed sin that
// each is multiplied with.  y = x cos + partner * sn, where sn carries the
// sign of the sum's second term.
struct Turn {
    float2 cs[4], sn[4];
    bool any;  // one of the eight is rotated
    int src;   // kShuffle: the partners' lane
};

template <int PAIRS>
__device__ __forceinline__ void load_turn(const Rotary &r, int64_t pos, int c, Turn &t) {
    const int half = r.dim >> 1, lane = threadIdx.x & 31;
    const float sign = (r.flags & OQ_ROTARY_INVERSE) ? -1.0f : 1.0f;
    const float *row = r.table + pos * r.dim;
    t.any = 8 * c < r.dim;
    if (PAIRS == kShuffle) {
        t.src = !t.any ? lane : (8 * c < half ? lane + (half >> 3) : lane - (half >> 3));
        if (t.any) {
            const int i0 = 8 * c < half ? 8 * c : 8 * c - half;
            const float s = 8 * c < half ? -sign : sign;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float4 a = __ldg(reinterpret_cast<const float4 *>(row + i0) + q);
                const float4 b = __ldg(reinterpret_cast<const float4 *>(row + half + i0) + q);
                t.cs[2 * q] = make_float2(a.x, a.y), t.cs[2 * q + 1] = make_float2(a.z, a.w);
                t.sn[2 * q] = make_float2(s * b.x, s * b.y), t.sn[2 * q + 1] = make_float2(s * b.z, s * b.w);
            }
        }
        return;
    }
    if (PAIRS == kNext) {
        if (t.any) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(row + 4 * c));
            const float4 b = __ldg(reinterpret_cast<const float4 *>(row + half + 4 * c));
            const float cs[4] = {a.x, a.y, a.z, a.w}, sn[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                t.cs[e] = make_float2(cs[e], cs[e]);
                t.sn[e] = make_float2(-sign * sn[e], sign * sn[e]);
            }
        }
        return;
    }
    const bool inter = r.flags & OQ_ROTARY_INTERLEAVED;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int i = 8 * c + e;
        float cs = 1.0f, sn = 0.0f;
        if (i < r.dim) {
            const int a = inter ? i >> 1 : (i < half ? i : i - half);
            const bool first = inter ? !(i & 1) : i < half;
            cs = __ldg(row + a);
            sn = (first ? -sign : sign) * __ldg(row + half + a);
        }
        (e & 1 ? t.cs[e >> 1].y : t.cs[e >> 1].x) = cs;
        (e & 1 ? t.sn[e >> 1].y : t.sn[e >> 1].x) = sn;
    }
}

// x cos -+ partner sin of two elements, each product and the sum rounded to
// fp32: the same bits as the formula in separate operations.  The packed
// multiply and add would be joined into one fused operation even where both
// are stated as rounding, so the sum is a product with `one` plus the other
// term: 1.0f from the kernel's arguments, which the compiler does not know.
__device__ __forceinline__ float2 turn2(float2 x, float2 cs, float2 partner, float2 sn, float one) {
    return __ffma2_rn(__fmul2_rn(x, cs), make_float2(one, one), __fmul2_rn(partner, sn));
}

// Rotates a lane's eight elements.  All lanes of the warp take part; `row` is
// the head's first element (nullptr: no head).
template <typename T, int PAIRS>
__device__ __forceinline__ void rotate8(const Rotary &r, const Turn &t, const T *row, int c, float2 (&x)[4]) {
    if (PAIRS == kShuffle) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float2 p;
            p.x = __shfl_sync(0xffffffffu, x[e].x, t.src);
            p.y = __shfl_sync(0xffffffffu, x[e].y, t.src);
            if (t.any) x[e] = turn2(x[e], t.cs[e], p, t.sn[e], r.one);
        }
        return;
    }
    if (!t.any) return;
    if (PAIRS == kNext) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = turn2(x[e], t.cs[e], make_float2(x[e].y, x[e].x), t.sn[e], r.one);
        return;
    }
    const int half = r.dim >> 1;
    const bool inter = r.flags & OQ_ROTARY_INTERLEAVED;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = 8 * c + 2 * e;
        float2 p = make_float2(x[e].y, x[e].x);
        if (!inter) {
            p = make_float2(0.0f, 0.0f);
            if (row != nullptr && i < r.dim) p.x = Elem<T>::to_f32(row[i < half ? i + half : i - half]);
            if (row != nullptr && i + 1 < r.dim) p.y = Elem<T>::to_f32(row[i + 1 < half ? i + 1 + half : i + 1 - half]);
        }
        const float2 y = turn2(x[e], t.cs[e], p, t.sn[e], r.one);
        if (i < r.dim) x[e].x = y.x;  // an unrotated element keeps its bits
        if (i + 1 < r.dim) x[e].y = y.y;
    }
}

// ------------------------------------------------------------- rotary ----
//
// HBM bound: every element is read and written once and needs 3 flops.  A
// lane owns eight consecutive elements of a head (16 bytes of a 16-bit type),
// head_dim / 8 lanes a head; a round is the 32 * 8 / head_dim heads that a
// warp takes at once.  A warp walks rounds of ONE token with kRows of them in
// flight: the token's cos and sin are loaded once into registers for all of
// them, and the partner of an element comes from another lane by shuffle (half
// layout) or is the lane's own neighbour (interleaved).
// 8192 tokens x 64 heads x 128, bf16: 45 us, 6.0 TB/s, 92 % of the measured copy
// rate (69 us with one step of four rounds a warp: each then waits for its
// position and table row by itself).  2049 x 40 x 128 fp32, 64 of them rotated
// interleaved: 16 us, 83 %.
template <typename T, bool VEC, int PAIRS>
__global__ void __launch_bounds__(kWarps * 32)
rotary_kernel(Rows x, T *y, int64_t y_ts, int64_t y_hs, int64_t tokens, int heads, int head_dim, Rotary rot,
              int parts, int rounds) {
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int64_t t = unit / parts;
    if (t >= tokens) return;
    const int lpr = head_dim >> 3, per = 32 / lpr;  // lanes a head, heads a round
    const int sub = lane / lpr, c = lane - sub * lpr;
    const int round0 = (int)(unit - t * parts) * rounds;
    const T *xt = static_cast<const T *>(x.p) + t * x.ts;
    // this lane's heads: every per-th from h on, n of them
    const int h = round0 * per + sub, end = min((round0 + rounds) * per, heads);
    const int n = sub < per && h < end ? (end - h + per - 1) / per : 0;
    const int steps = min(rounds, (heads + per - 1) / per - round0);  // of the warp
    const T *src = xt + h * x.hs + 8 * c;
    T *dst = y + t * y_ts + h * y_hs + 8 * c;
    const int64_t x_step = per * x.hs, y_step = per * y_hs;
    Eight<T> next[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
        if (i < n) load_row8<T, VEC>(src + i * x_step, next[i]);
    const int64_t pos = position_at(rot, t);
    const bool ok = pos >= 0 && pos < rot.rows;
    if (!ok && lane == 0) index_error();
    Turn turn;
    load_turn<PAIRS>(rot, ok ? pos : 0, c, turn);
    for (int s = 0; s < steps; s += kRows) {
        const T *ahead = src + kRows * x_step;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (s + i >= steps) break;
            float2 v[4];
            widen(next[i], v);
            if (s + i + kRows < n) load_row8<T, VEC>(ahead, next[i]);
            const bool in = s + i < n;
            rotate8<T, PAIRS>(rot, turn, in ? src - 8 * c : nullptr, c, v);
            if (PAIRS == kAny) __syncwarp();  // y may be x: partners are read before any store of the warp
            if (ok && in) store_row8<T, VEC>(dst, v);
            src += x_step, ahead += x_step, dst += y_step;
        }
    }
}

// Place of the step's token t in its sequence, and its row of head 0 in the
// cache (-1: none).  Returns false for a padding token, and with an error for
// one of a sequence whose starts are not in order.
__device__ __forceinline__ bool find_row(const Batch &bt, int seq, int64_t t, int64_t tokens, int64_t pages,
                                         int page_size, int kv_heads, int64_t &pos, int64_t &at) {
    if (seq >= bt.sequences) return false;
    int first, count;
    if (!tokens_of(bt, seq, tokens, first, count) || t < first || t >= first + count) {
        if ((threadIdx.x & 31) == 0) index_error();
        return false;
    }
    // The place that the length gives, inside the page-table row or not: a
    // length cut to the row would move the tokens onto others that are there.
    pos = (int64_t)__ldg(bt.lengths + seq) - count + (t - first);
    if (pos >= 0 && pos < (int64_t)bt.max_pages * page_size) {
        const int p = (int)pos, slot = p / page_size, page = __ldg(bt.table + (int64_t)seq * bt.max_pages + slot);
        if (page >= 0 && page < pages) at = ((int64_t)page * kv_heads) * page_size + (p - slot * page_size);
    }
    if (at < 0 && (threadIdx.x & 31) == 0) index_error();
    return true;
}

// The codes of eight elements as a word: clip(rint(fl(x / s)), -7, 7) with
// fl() the IEEE quotient.  r = x * rcp(s) is within 2e-6 of it where the
// clipped range is not left, so both round to the same integer unless r is
// within 1e-5 of a half; then (2 in 10^5), and beyond the range, the word
// takes the divisions.  (A scale is at least max / 7 (1 - 2^-8), so r leaves
// [-7.04, 7.04] only where the scale was limited, or is an fp16 subnormal.)
// Adding 1.5 * 2^23 + 8 leaves u = code + 8 in the low
// bits of 0x4B400000 + u; the eight sums shifted by 4 e add up, and the
// constants' own sum is 0x3F400000 (mod 2^32).
constexpr float kMagic = kRoundMagic + 8.0f;

__device__ __noinline__ uint32_t divide8(float2 x0, float2 x1, float2 x2, float2 x3, float s) {
    const float x[8] = {x0.x, x0.y, x1.x, x1.y, x2.x, x2.y, x3.x, x3.y};
    uint32_t acc = 0;
#pragma unroll
    for (int e = 7; e >= 0; --e)
        acc = acc * 16 + __float_as_uint(__fadd_rn(fminf(fmaxf(rintf(__fdiv_rn(x[e], s)), -7.0f), 7.0f), kMagic));
    return acc;
}

// mx: the group's largest magnitude.
__device__ __forceinline__ uint32_t pack8(const float2 (&x)[4], float s, float mx) {
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    const float2 inv2 = make_float2(inv, inv), up = make_float2(kMagic, kMagic), down = make_float2(-kMagic, -kMagic);
    uint32_t acc = 0;
    float off = 0.0f;  // the largest distance from an integer
#pragma unroll
    for (int e = 3; e >= 0; --e) {
        const float2 r = __fmul2_rn(x[e], inv2), t = __fadd2_rn(r, up), n = __fadd2_rn(t, down);
        const float2 d = __fadd2_rn(r, make_float2(-n.x, -n.y));
        off = fmaxf(off, fmaxf(fabsf(d.x), fabsf(d.y)));
        acc = (acc * 16 + __float_as_uint(t.y)) * 16 + __float_as_uint(t.x);
    }
    if (off > 0.49999f || mx > 7.4f * s) acc = divide8(x[0], x[1], x[2], x[3], s);
    return (acc - 0x3F400000u) ^ 0x88888888u;
}

// A group's scale: fl(mx / 7) (Markstein's correction of the product with
// RN(1 / 7), the IEEE quotient of every positive finite mx), 8 bits, fp16.
__device__ __forceinline__ float scale_of(float mx) {
    const float y = 0.14285714924335479736f, q = __fmul_rn(mx, y);
    const float s = fmaf(fmaf(-q, 7.0f, mx), y, q);
    const float s16 = fminf(__half2float(__float2half_rn(__bfloat162float(__float2bfloat16_rn(s)))), kMaxScale);
    return s16 == 0.0f ? 1.0f : s16;
}

// ------------------------------------------------------------- append ----
//
// HBM bound at many tokens, latency bound at a few.  The same lane layout and
// walk as the rotary kernel, over the token's query heads and then its key
// and value heads in pairs (k0 v0 k1 v1 ...), so that a key and the value that
// goes with it sit in neighbouring lane groups of one round.  A group's
// maximum is a shuffle over group / 8 lanes; a lane's eight codes are one word.
// 7622 tokens of 32 query and 32 key heads x 128, fp16, rotated: 90 us against
// 44 us of HBM time.  ncu: issue 64 %, 158 instructions a round of two heads,
// DRAM 36 % -- instruction-bound: two roundings and a shuffle an element for the
// rotation, six operations an element for the codes.  (It took 300 us with the
// queries', keys' and values' rows in one loop, a maximum that propagates NaN
// by comparisons, and a division per element near a tie of 0.1 %.)
struct AppendArgs {
    Rows q, k, v;
    void *q_out;
    int64_t qo_ts, qo_hs;
    int q_heads, kv_heads, page_size, group_log;  // log2(group / 8): lanes a group
    uint32_t *k_codes, *v_codes;
    __half *k_scales, *v_scales;
    int64_t pages, tokens;
    int parts, rounds, q_rounds, all_rounds;  // rounds a warp; of the queries; of a token
    Rotary rot;                               // table nullptr: no rotation
    Batch batch;
};

template <typename T, int D, bool VEC, int PAIRS>
__global__ void __launch_bounds__(kWarps * 32, VEC && PAIRS != kAny ? 6 : 1) append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int LPR = D / 8, PER = 32 / LPR;
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int64_t t = unit / a.parts;
    if (t >= a.tokens) return;
    const int sub = lane / LPR, c = lane % LPR;
    const int round0 = (int)(unit - t * a.parts) * a.rounds, round1 = min(round0 + a.rounds, a.all_rounds);

    // Rounds [round0, q1) are the queries': the lane's head is round * PER +
    // sub.  Rounds [kv0, ...) (counted from the first one after the queries)
    // are the keys' and values': a lane group has keys only or values only.
    const int q1 = PAIRS != kNone ? min(round1, a.q_rounds) : 0;
    const int q_steps = max(q1 - round0, 0), qh = round0 * PER + sub;
    const int q_n = q_steps > 0 && qh < a.q_heads ? min(q_steps, (a.q_heads - qh + PER - 1) / PER) : 0;
    const int kv0 = max(round0 - a.q_rounds, 0), kv_steps = max(round1 - a.q_rounds - kv0, 0);
    const int kvh = kv0 * (PER / 2) + (sub >> 1);
    const int kv_n = kvh < a.kv_heads ? min(kv_steps, (a.kv_heads - kvh + PER / 2 - 1) / (PER / 2)) : 0;
    const bool is_v = sub & 1;
    const Rows &kv = is_v ? a.v : a.k;
    const int64_t q_step = PER * a.q.hs, kv_step = (PER / 2) * kv.hs;
    const T *q_src = static_cast<const T *>(a.q.p) + t * a.q.ts + qh * a.q.hs + 8 * c;
    const T *kv_src = static_cast<const T *>(kv.p) + t * kv.ts + kvh * kv.hs + 8 * c;
    Eight<T> next[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (q_steps > 0) {
            if (i < q_n) load_row8<T, VEC>(q_src + i * q_step, next[i]);
        } else if (i < kv_n) {
            load_row8<T, VEC>(kv_src + i * kv_step, next[i]);
        }
    }

    const int seq = sequence_of(a.batch, (int)t);
    int64_t pos = 0, at = -1;  // place in the sequence; row of head 0 in the cache
    const bool real = find_row(a.batch, seq, t, a.tokens, a.pages, a.page_size, a.kv_heads, pos, at);
    const int64_t angle = PAIRS != kNone && a.rot.positions != nullptr ? position_at(a.rot, t) : pos;
    const bool ok = PAIRS == kNone || (angle >= 0 && angle < a.rot.rows);
    if (!ok && real && lane == 0) index_error();
    Turn turn;
    if (PAIRS != kNone) load_turn<PAIRS>(a.rot, ok ? angle : 0, c, turn);

    // ---- queries (only with a rotation)
    if (q_steps > 0) {
        T *dst = static_cast<T *>(a.q_out) + t * a.qo_ts + qh * a.qo_hs + 8 * c;
        const int64_t out_step = PER * a.qo_hs;
        for (int s = 0; s < q_steps; s += kRows) {
            const T *ahead = q_src + kRows * q_step;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                if (s + i >= q_steps) break;
                float2 x[4];
                widen(next[i], x);
                if (s + i + kRows < q_n) load_row8<T, VEC>(ahead, next[i]);
                const bool in = s + i < q_n;
                rotate8<T, PAIRS>(a.rot, turn, in ? q_src - 8 * c : nullptr, c, x);
                if (PAIRS == kAny) __syncwarp();  // q_out may be q: partners are read before any store of the warp
                if (ok && in) store_row8<T, VEC>(dst, x);
                q_src += q_step, ahead += q_step, dst += out_step;
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (i < kv_n) load_row8<T, VEC>(kv_src + i * kv_step, next[i]);
    }

    // ---- keys and values
    if (PAIRS != kNone) turn.any = turn.any && !is_v;
    const unsigned pair = (LPR == 16 ? 0xffffffffu : 0xffffu) << ((sub >> 1) * 2 * LPR % 32);
    const int groups = LPR >> a.group_log;
    const bool put = at >= 0 && ok, first = put && (c & ((1 << a.group_log) - 1)) == 0;
    const int64_t row = at + (int64_t)kvh * a.page_size;
    uint32_t *codes = (is_v ? a.v_codes : a.k_codes) + row * (D / 8) + c;
    __half *scales = (is_v ? a.v_scales : a.k_scales) + row * groups + (c >> a.group_log);
    const int64_t code_step = (int64_t)(PER / 2) * a.page_size * (D / 8);
    const int64_t scale_step = (int64_t)(PER / 2) * a.page_size * groups;
    for (int s = 0; s < kv_steps; s += kRows) {
        const T *ahead = kv_src + kRows * kv_step;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (s + i >= kv_steps) break;  // warp-uniform
            float2 x[4];
            widen(next[i], x);
            if (s + i + kRows < kv_n) load_row8<T, VEC>(ahead, next[i]);
            const bool in = s + i < kv_n;
            if (PAIRS != kNone) rotate8<T, PAIRS>(a.rot, turn, in ? kv_src - 8 * c : nullptr, c, x);
            float mx = 0.0f;
            float2 nan = make_float2(0.0f, 0.0f);  // 0 * x: NaN where x is not finite
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                mx = fmaxf(mx, fmaxf(fabsf(x[e].x), fabsf(x[e].y)));
                nan = __ffma2_rn(x[e], make_float2(0.0f, 0.0f), nan);
            }
            // Not finite anywhere in the token's key or value of this head: the
            // lanes of both (2 * LPR of them) agree on it.
            const bool bad = (__ballot_sync(0xffffffffu, in && !(nan.x + nan.y == 0.0f)) & pair) != 0;
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (a.group_log > 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            if (a.group_log > 3) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            const float sc = bad ? 1.0f : scale_of(mx);
            uint32_t word = pack8(x, sc, bad ? 0.0f : mx);
            if (bad) word = 0;
            if (put && in) *codes = word;
            if (first && in) *scales = bad && !is_v ? __ushort_as_half(0x7FFF) : __float2half_rn(sc);
            kv_src += kv_step, ahead += kv_step, codes += code_step, scales += scale_step;
        }
    }
}

// --------------------------------------------------------------- read ----
//
// HBM bound; the walk of the append kernel over the key and value heads.  7622
// tokens of 32 heads x 128 to fp16: 30 us against 24 us of HBM time.
template <typename T>
__device__ __forceinline__ void values8(uint32_t word, __half scale, T (&o)[8]) {
    __half2 v[4];
    unpack_int(word, v);  // pairs (i, i + 4)
    const __half2 s = __half2half2(scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = __hmul2(v[i], s);  // exact
        if constexpr (std::is_same<T, __half>::value) {
            o[i] = __low2half(v[i]);
            o[i + 4] = __high2half(v[i]);
        } else {
            o[i] = from_f32<T>(__low2float(v[i]));
            o[i + 4] = from_f32<T>(__high2float(v[i]));
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32)
read_kernel(const uint32_t *k_codes, const __half *k_scales, const uint32_t *v_codes, const __half *v_scales, T *k,
            T *v, Batch batch, int64_t pages, int page_size, int kv_heads, int group_log, int64_t tokens, int parts,
            int rounds) {
    constexpr int LPR = D / 8, PER = 32 / LPR;
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int64_t t = unit / parts;
    if (t >= tokens) return;
    const int sub = lane / LPR, c = lane % LPR;
    const bool is_v = sub & 1;  // a lane group has keys only or values only
    const int seq = sequence_of(batch, (int)t);
    int64_t pos = 0, at = -1;
    find_row(batch, seq, t, tokens, pages, page_size, kv_heads, pos, at);
    const int round0 = (int)(unit - t * parts) * rounds, round1 = round0 + rounds;
    const int groups = LPR >> group_log;
    const int64_t base = at + (int64_t)(sub >> 1) * page_size;
    const uint32_t *codes = (is_v ? v_codes : k_codes) + base * (D / 8) + c;
    const __half *scales = (is_v ? v_scales : k_scales) + base * groups + (c >> group_log);
    T *dst = (is_v ? v : k) + (t * kv_heads + (sub >> 1)) * D + 8 * c;
    uint32_t next[kRows];
    __half scale[kRows];
    auto in = [&](int round) { return round < round1 && round * (PER / 2) + (sub >> 1) < kv_heads; };
    auto fetch = [&](int round) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            next[i] = 0;
            scale[i] = __ushort_as_half(0);
            if (at >= 0 && in(round + i)) {
                const int64_t row = (int64_t)((round + i) * (PER / 2)) * page_size;
                next[i] = codes[row * (D / 8)];
                scale[i] = scales[row * groups];
            }
        }
    };
    fetch(round0);
    for (int round = round0; round < round1 && round * (PER / 2) < kv_heads; round += kRows) {
        uint32_t word[kRows];
        __half s[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            word[i] = next[i];
            s[i] = scale[i];
        }
        fetch(round + kRows);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (!in(round + i)) continue;
            Eight<T> o;
            values8<T>(word[i], s[i], o.e);
#pragma unroll
            for (int x = 0; x < (int)sizeof(T) / 2; ++x)
                reinterpret_cast<uint4 *>(dst + (int64_t)((round + i) * (PER / 2)) * D)[x] =
                    reinterpret_cast<const uint4 *>(o.e)[x];
        }
    }
}

// Rounds a warp takes of a token that has `all`: as many as leave the GPU
// kFill warps a SM, in steps of kRows, at most `most`.  (Few: a warp's lookups
// are paid for more often; many: too few warps at small sizes, and a last
// wave of warps that leaves SMs idle.  Measured, 8 to 48 rounds: rotary of
// 8192 x 64 x 128 50 to 45 us, least at 16; append and read of 7622 tokens of
// 32 heads 158 to 136 us, flat from 24 on, where the lookups are a longer chain.)
constexpr int kFill = 32;

int rounds_of(int64_t tokens, int64_t all, int most) {
    const int64_t want = tokens * all / ((int64_t)sm_count() * kFill);
    const int64_t r = want / kRows * kRows;
    return (int)(r < kRows ? kRows : (r > most ? most : r));
}

int check_rotary(const oq_rotary_spec *r, int head_dim) {
    OQ_REQUIRE(r->table != nullptr && aligned(r->table, 16), "the rotary table must be a 16-byte aligned array");
    OQ_REQUIRE(r->rows >= 1, "the rotary table is empty");
    OQ_REQUIRE(r->dim >= 2 && r->dim % 2 == 0 && r->dim <= head_dim,
               "the rotary dimension must be even, at least 2 and at most head_dim");
    OQ_REQUIRE((r->flags & ~(OQ_ROTARY_INTERLEAVED | OQ_ROTARY_INVERSE)) == 0, "unknown rotary flags");
    return OQ_OK;
}

int grid_of(int64_t units, int64_t *blocks) {
    *blocks = cdiv(units, kWarps);
    OQ_REQUIRE(*blocks < (1ll << 31), "too many tokens and heads for one call");
    return OQ_OK;
}

template <typename T, bool VEC>
void rotary_start(const Rows &x, void *y, int64_t y_ts, int64_t y_hs, int64_t tokens, int heads, int head_dim,
                  const Rotary &rot, int parts, int rounds, unsigned blocks, cudaStream_t st) {
    const int pairs = pairs_of(rot);
    auto kern = pairs == kShuffle ? rotary_kernel<T, VEC, kShuffle>
                : pairs == kNext  ? rotary_kernel<T, VEC, kNext>
                                  : rotary_kernel<T, VEC, kAny>;
    kern<<<blocks, kWarps * 32, 0, st>>>(x, static_cast<T *>(y), y_ts, y_hs, tokens, heads, head_dim, rot, parts,
                                         rounds);
}

template <typename T>
int rotary_launch(const Rows &x, void *y, int64_t y_ts, int64_t y_hs, int64_t tokens, int heads, int head_dim,
                  const Rotary &rot, cudaStream_t st) {
    const int64_t all = cdiv(heads, 32 / (head_dim / 8));
    const int rounds = rounds_of(tokens, all, 16), parts = (int)cdiv(all, rounds);
    int64_t blocks;
    if (int rc = grid_of(tokens * parts, &blocks)) return rc;
    const int64_t n = 16 / sizeof(T);
    const bool vec = aligned(x.p, 16) && aligned(y, 16) && x.ts % n == 0 && x.hs % n == 0 && y_ts % n == 0 &&
                     y_hs % n == 0;
    (vec ? rotary_start<T, true> : rotary_start<T, false>)(x, y, y_ts, y_hs, tokens, heads, head_dim, rot, parts,
                                                           rounds, (unsigned)blocks, st);
    return check_launch("rotary");
}

template <typename T, int D, bool VEC>
void append_start(const AppendArgs &a, unsigned blocks, cudaStream_t st) {
    const int pairs = pairs_of(a.rot);
    auto kern = pairs == kNone      ? append_kernel<T, D, VEC, kNone>
                : pairs == kShuffle ? append_kernel<T, D, VEC, kShuffle>
                : pairs == kNext    ? append_kernel<T, D, VEC, kNext>
                                    : append_kernel<T, D, VEC, kAny>;
    kern<<<blocks, kWarps * 32, 0, st>>>(a);
}

template <typename T, int D>
int append_launch(const AppendArgs &a, bool vec, int64_t blocks, cudaStream_t st) {
    (vec ? append_start<T, D, true> : append_start<T, D, false>)(a, (unsigned)blocks, st);
    return check_launch("kv4_append");
}

template <typename T, int D>
int read_launch(const oq_kv4_cache *c, const Batch &b, void *k, void *v, int group_log, int64_t tokens, int parts,
                int rounds, int64_t blocks, cudaStream_t st) {
    read_kernel<T, D><<<(unsigned)blocks, kWarps * 32, 0, st>>>(
        reinterpret_cast<const uint32_t *>(c->k_codes), static_cast<const __half *>(c->k_scales),
        reinterpret_cast<const uint32_t *>(c->v_codes), static_cast<const __half *>(c->v_scales), static_cast<T *>(k),
        static_cast<T *>(v), b, c->pages, c->page_size, c->kv_heads, group_log, tokens, parts, rounds);
    return check_launch("kv4_read");
}

int group_log_of(int group) { return group == 32 ? 2 : group == 64 ? 3 : 4; }

}  // namespace
}  // namespace kv4
}  // namespace oq

using namespace oq;
using namespace oq::kv4;

extern "C" int oq_rotary(const void *x, void *y, int dtype, int64_t tokens, int heads, int head_dim,
                         int64_t x_token_stride, int64_t x_head_stride, int64_t y_token_stride, int64_t y_head_stride,
                         const oq_rotary_spec *rotary, const void *positions, int positions_64, oq_stream_t stream) {
    clear_error();
    OQ_REQUIRE(dtype == OQ_F32 || dtype == OQ_F16 || dtype == OQ_BF16, "rotary: x must be fp32, fp16 or bf16");
    OQ_REQUIRE(tokens >= 1 && heads >= 1, "rotary: dimensions must be positive");
    OQ_REQUIRE(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0,
               "rotary: head_dim must be a multiple of 8 up to 256");
    OQ_REQUIRE(x && y && rotary && positions, "null pointer argument");
    if (int rc = check_rotary(rotary, head_dim)) return rc;
    const Rows r{x, x_token_stride, x_head_stride};
    const Rotary rot{rotary->table, rotary->rows, rotary->dim, rotary->flags, positions, positions_64};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == OQ_F32)
        return rotary_launch<float>(r, y, y_token_stride, y_head_stride, tokens, heads, head_dim, rot, st);
    if (dtype == OQ_F16)
        return rotary_launch<__half>(r, y, y_token_stride, y_head_stride, tokens, heads, head_dim, rot, st);
    return rotary_launch<__nv_bfloat16>(r, y, y_token_stride, y_head_stride, tokens, heads, head_dim, rot, st);
}

extern "C" int oq_kv4_append(const oq_kv4_cache *cache, const oq_kv4_batch *batch, const void *q, void *q_out,
                             int q_heads, int64_t q_token_stride, int64_t q_head_stride, int64_t qo_token_stride,
                             int64_t qo_head_stride, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                             const void *v, int64_t v_token_stride, int64_t v_head_stride, int dtype, int64_t tokens,
                             const oq_rotary_spec *rotary, const void *positions, int positions_64,
                             oq_stream_t stream) {
    clear_error();
    OQ_REQUIRE(dtype == OQ_F16 || dtype == OQ_BF16, "kv4_append: k and v must be fp16 or bf16");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(batch, tokens)) return rc;
    OQ_REQUIRE(k && v, "null pointer argument");
    OQ_REQUIRE(q == nullptr || (q_out != nullptr && q_heads >= 1), "kv4_append: q needs q_out and its head count");
    OQ_REQUIRE(rotary != nullptr || (q == nullptr && positions == nullptr),
               "kv4_append: q and positions need a rotary table");
    if (rotary != nullptr)
        if (int rc = check_rotary(rotary, cache->head_dim)) return rc;
    AppendArgs a = {};
    a.q = Rows{q, q_token_stride, q_head_stride};
    a.k = Rows{k, k_token_stride, k_head_stride};
    a.v = Rows{v, v_token_stride, v_head_stride};
    a.q_out = q_out;
    a.qo_ts = qo_token_stride;
    a.qo_hs = qo_head_stride;
    a.q_heads = q != nullptr ? q_heads : 0;
    a.kv_heads = cache->kv_heads;
    a.page_size = cache->page_size;
    a.group_log = group_log_of(cache->group_size);
    a.k_codes = reinterpret_cast<uint32_t *>(cache->k_codes);
    a.v_codes = reinterpret_cast<uint32_t *>(cache->v_codes);
    a.k_scales = static_cast<__half *>(cache->k_scales);
    a.v_scales = static_cast<__half *>(cache->v_scales);
    a.pages = cache->pages;
    a.tokens = tokens;
    const int per = 32 / (cache->head_dim / 8);
    a.q_rounds = (int)cdiv(a.q_heads, per);
    a.all_rounds = a.q_rounds + (int)cdiv(2 * a.kv_heads, per);
    a.rounds = rounds_of(tokens, a.all_rounds, 32);
    a.parts = (int)cdiv(a.all_rounds, a.rounds);
    if (rotary != nullptr)
        a.rot = Rotary{rotary->table, rotary->rows, rotary->dim, rotary->flags, positions, positions_64};
    a.batch = device_batch(batch);
    auto ok = [](const void *p, int64_t ts, int64_t hs) { return aligned(p, 16) && ts % 8 == 0 && hs % 8 == 0; };
    const bool vec = ok(k, k_token_stride, k_head_stride) && ok(v, v_token_stride, v_head_stride) &&
                     (q == nullptr || (ok(q, q_token_stride, q_head_stride) &&
                                       ok(q_out, qo_token_stride, qo_head_stride)));
    int64_t blocks;
    if (int rc = grid_of(tokens * a.parts, &blocks)) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == OQ_F16)
        return cache->head_dim == 64 ? append_launch<__half, 64>(a, vec, blocks, st)
                                     : append_launch<__half, 128>(a, vec, blocks, st);
    return cache->head_dim == 64 ? append_launch<__nv_bfloat16, 64>(a, vec, blocks, st)
                                 : append_launch<__nv_bfloat16, 128>(a, vec, blocks, st);
}

extern "C" int oq_kv4_read(const oq_kv4_cache *cache, const oq_kv4_batch *batch, void *k, void *v, int dtype,
                           int64_t tokens, oq_stream_t stream) {
    clear_error();
    OQ_REQUIRE(dtype == OQ_F32 || dtype == OQ_F16 || dtype == OQ_BF16, "kv4_read: output must be fp32, fp16 or bf16");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(batch, tokens)) return rc;
    OQ_REQUIRE(k && v, "null pointer argument");
    OQ_REQUIRE(aligned(k, 16) && aligned(v, 16), "kv4_read: k and v must be 16-byte aligned");
    const int per = 32 / (cache->head_dim / 8);
    const int64_t all = cdiv(2 * cache->kv_heads, per);
    const int rounds = rounds_of(tokens, all, 32), parts = (int)cdiv(all, rounds);
    int64_t blocks;
    if (int rc = grid_of(tokens * parts, &blocks)) return rc;
    const int gl = group_log_of(cache->group_size);
    const Batch b = device_batch(batch);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool d64 = cache->head_dim == 64;
    if (dtype == OQ_F32)
        return d64 ? read_launch<float, 64>(cache, b, k, v, gl, tokens, parts, rounds, blocks, st)
                   : read_launch<float, 128>(cache, b, k, v, gl, tokens, parts, rounds, blocks, st);
    if (dtype == OQ_F16)
        return d64 ? read_launch<__half, 64>(cache, b, k, v, gl, tokens, parts, rounds, blocks, st)
                   : read_launch<__half, 128>(cache, b, k, v, gl, tokens, parts, rounds, blocks, st);
    return d64 ? read_launch<__nv_bfloat16, 64>(cache, b, k, v, gl, tokens, parts, rounds, blocks, st)
               : read_launch<__nv_bfloat16, 128>(cache, b, k, v, gl, tokens, parts, rounds, blocks, st);
}
