// Attention over the 4-bit key/value cache, queries of a few rows per key
// head: the cache is streamed once and multiplied on mma.sync.
//
// Mathematics.  For a key head, its query rows (tokens of the step x query
// heads of the key head) are columns n of small products.  A warp takes 16
// cached tokens at a time:
//     c_G[t][n] = sum over d in group G of code_k[t][d] q[n][d]     (integers exact in fp16, fp32 sums)
//     s[t][n]   = sum_G scale_k[t][G] c_G[t][n]                     (fp32)
//     p         = 2^(s f - m)          f = scale log2 e, m a running maximum of the column
//     o[d][n]  += sum_t (code_v[t][d] scale_v[t][G]) p[t][n]        (cached values exact in fp16)
// and columns end as o / sum p.  p is the only rounding before the output's:
// to fp16, 11 bits, with m kept 6 below the maximum seen so that p sits in
// [2^-24, 2^14] and small weights keep their bits.  A warp raises m only when
// a score passes m + 14 (a warp vote per 16 tokens), which is rare after the
// first tokens, so the maximum costs no shuffles in the steady state.
//
// Queries in bf16 go to fp16 times a power of two per row (fp16_power): one
// kernel for both types.
//
// What bounds it.  The cache has to be read once: 144 bytes a token and key
// head (head_dim 128, groups of 32).  64 ragged sequences of 333 to 8192 tokens
// (64 query, 8 key heads): 81.6 us, 59 % of the measured copy rate, DRAM traffic
// 1.00 x the cache's bytes; two of 100003 and 131071 tokens (groups of 64) 65
// us, 59 %.  ncu: instruction issue 62 % of the cycles with 12 warps an SM, 22
// instructions a token and key head, most of them the unpacking (9 for eight
// codes, and 4 more for the scale of V); no bank conflicts, tensor pipe 22 %.
// So it is bound by issue and by the latency of what each warp does in turn.
// Fewer warps are slower (8 an SM: 122 us) and more do not have the registers
// (16: 88 us with one block a step, 86 us with two and spills; 20: 117 us).
// Deeper rings (6 stages: 82.8 us) and scores computed a step ahead (85 us) cost
// more than they hide.
#include <climits>

#include "oq_kv4_attention.cuh"

namespace oq {
namespace kv4 {
namespace {

constexpr int kWarps = 4;   // warps a CTA; each works by itself
// CTAs an SM: three leave 168 registers a thread.  With four, 128, the loop
// spills: 64 ragged sequences 86 us for 83.  Two tiles of columns of head_dim
// 128 hold 64 more sums and need two CTAs: 16 rows on 16 x 8000 tokens 62 us for
// 66, on 8 x 4000 tokens of 32 key heads 62 for 65.
template <int HD, int NT>
constexpr int kCtas = NT == 2 && HD == 128 ? 2 : 3;
constexpr int kStages = 4;  // 16-token stages of a warp, in use or in flight
// Cost of beginning an item and the smallest share of a warp, in blocks of 16
// tokens.  Measured with 8, 12, 14 and 4 .. 40: 64 ragged sequences 83.2 / 81.6 /
// 82.2 us for the first; one sequence of 1000 tokens and 32 key heads 12 us with a
// least share of 4, 29 us with 40.
constexpr int kSetup = 12, kLeast = 4;

using Args = AttnArgs;

// A partial result: m[cols], l[cols], then o as the lanes hold it (float4
// [NT * HD / 16][32 lanes]: coalesced, and the joining kernel has the same lanes).
template <int HD, int NT>
struct Shape {
    static constexpr int kCols = 8 * NT;
    static constexpr int kSlices = NT * HD / 16;
    static constexpr int kPart = 2 * kCols + kSlices * 128;
    static constexpr int kPitch = HD / 2 + 16;  // bytes of a staged row: 16-byte steps over all banks
};

// Work of sequence b: an item per key head and per block of `cols` query
// rows, of nb blocks of 16 cached tokens (from block b0 on) and kSetup units.
struct Work {
    int first, count, rows;
    int length, base;  // cached tokens that can be read; position of the step's first token
    int floor;         // first cached token any row sees
    int b0, nb, blocks;
    bool out;  // left out: no blocks, and its rows are cleared by the joining kernel
};

__device__ __forceinline__ Work work_of(const Args &a, int b, int cols) {
    Work w;
    w.out = !tokens_of(a.batch, b, a.tokens, w.first, w.count) || w.count > a.max_tokens;
    int end;
    w.length = length_of(a.batch, b, a.page_size, end);
    w.base = end - w.count;
    w.rows = w.count * a.ratio;
    w.blocks = w.rows > a.few || w.out ? 0 : (w.rows + cols - 1) / cols;
    w.floor = a.window > 0 ? (int)max((int64_t)w.base + 1 - a.window, (int64_t)0) : 0;
    w.b0 = w.floor >> 4;
    w.nb = max(((w.length + 15) >> 4) - w.b0, 1);
    return w;
}

// Warps that share `all` units.
__device__ __forceinline__ int64_t shares_of(int64_t all, int warps) {
    const int64_t n = (all + kLeast - 1) / kLeast;
    return n < warps ? (n > 0 ? n : 1) : warps;
}

// Units before each sequence, and all of them: prefix[0 .. sequences] in shared
// memory, by the CTA's THREADS threads.
template <int THREADS>
__device__ __forceinline__ void units_before(const Args &a, int cols, int64_t *prefix) {
    __shared__ int64_t warp_sum[THREADS / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int64_t base = 0;
    for (int b0 = 0; b0 < a.batch.sequences; b0 += THREADS) {
        const int b = b0 + tid;
        int64_t n = 0;
        if (b < a.batch.sequences) {
            const Work w = work_of(a, b, cols);
            n = (int64_t)(w.nb + kSetup) * w.blocks * a.kv_heads;
        }
        int64_t inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) warp_sum[warp] = inc;
        __syncthreads();
        int64_t before = base;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += warp_sum[w];
            base += warp_sum[w];
        }
        if (b < a.batch.sequences) prefix[b] = before + inc - n;
        __syncthreads();
    }
    if (tid == 0) prefix[a.batch.sequences] = base;
    __syncthreads();
}

// x / y for y > 0, in 32 bits where that does (the usual case; 64-bit
// divisions are a hundred instructions).
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
    return ((x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with a zero accumulator to begin with (no registers to clear).
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Writes a warp's columns of an item: sums reduced over the lanes already, o
// divided by them.
template <typename T, int HD>
__device__ __forceinline__ void write_slice(const Args &a, const Work &w, int head, int col, int d, float x, float y,
                                            float m, float l) {
    if (col >= w.rows) return;
    const int tk = col / a.ratio;
    const int64_t row = (int64_t)(w.first + tk) * a.q_heads + head * a.ratio + (col - tk * a.ratio);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *dst = static_cast<T *>(a.out) + row * HD + d;
    put(dst, x * inv);
    put(dst + 1, y * inv);
    if (d == 0 && a.log_sum != nullptr) a.log_sum[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Every warp takes an equal share of all blocks of all items, one after the
// other: ragged lengths load the warps alike, and no warp waits for another.
// A share begins and ends inside an item, whose parts the joining kernel adds
// in a fixed order.  A warp streams its blocks through its own ring of cp.async
// stages, two blocks at a time (two independent chains of products; with one,
// 16 rows on 16 x 8000 tokens take 62.3 us for 59.6).  Rows are staged 16 bytes
// longer than they are, which makes both the ldmatrix of the keys and the 4- or
// 8-byte reads of the values free of bank conflicts.
template <typename T, int HD, int GS, int NT>
__global__ void __launch_bounds__(kWarps * 32, kCtas<HD, NT>) stream_kernel(const Args a) {
    using S = Shape<HD, NT>;
    constexpr int kCols = S::kCols, kPitch = S::kPitch;
    constexpr int NG = HD / GS;             // groups a row
    constexpr int CH = HD / 32;             // 16-byte chunks a row
    constexpr int kCodes = 16 * kPitch;     // staged codes of 16 tokens
    constexpr int kScales = 16 * NG * 2;
    constexpr int kStage = 2 * kCodes + 2 * kScales;
    constexpr int H = 2;                    // blocks a step
    constexpr int kSteps = kStages / H;     // steps in flight or in use
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    unsigned char *ring = smem + warp * kStages * kStage;
    const uint32_t ring_u = smem_u32(ring);
    // this lane's 16 bytes of a block of codes (or of scales: keys', then
    // values'), and where they are staged
    const uint8_t *k_lane = a.k_codes + lane * 16, *v_lane = a.v_codes + lane * 16;
    const unsigned char *sc_lane =
        reinterpret_cast<const unsigned char *>(lane < 2 * NG ? a.k_scales : a.v_scales) + lane % (2 * NG) * 16;
    const uint32_t to_codes = lane / CH * kPitch + lane % CH * 16;
    int64_t *prefix = reinterpret_cast<int64_t *>(smem + kWarps * kStages * kStage);
    asm volatile("griddepcontrol.launch_dependents;");

    units_before<kWarps * 32>(a, kCols, prefix);

    // Padding tokens: 0, log-sum -inf.
    {
        const int used = a.batch.starts != nullptr ? __ldg(a.batch.starts + a.batch.sequences) : a.batch.sequences;
        const int64_t row1 = a.tokens * a.q_heads;
        int64_t row = min((int64_t)max(used, 0), a.tokens) * a.q_heads + (int64_t)blockIdx.x * kWarps + warp;
        for (; row < row1; row += (int64_t)gridDim.x * kWarps) {
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) put(static_cast<T *>(a.out) + row * HD + i * 32 + lane, 0.0f);
            if (lane == 0 && a.log_sum != nullptr) a.log_sum[row] = -INFINITY;
        }
    }

    const int64_t all = prefix[a.batch.sequences];
    const int64_t shares = shares_of(all, gridDim.x * kWarps);
    const int64_t me = (int64_t)warp * gridDim.x + blockIdx.x;  // neighbouring shares on different SMs
    if (me >= shares) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // see the end
        return;
    }
    const int64_t u0 = quotient(me * all, shares), u1 = quotient((me + 1) * all, shares);

    for (int64_t u = u0; u < u1;) {
        // ---- the item of unit u
        int b;
        {
            int lo = 0, hi = a.batch.sequences;  // prefix[lo] <= u < prefix[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (prefix[mid] <= u)
                    lo = mid;
                else
                    hi = mid;
            }
            b = lo;
        }
        const Work w = work_of(a, b, kCols);
        const int64_t local = u - prefix[b];
        const int per = w.nb + kSetup, item = (int)quotient(local, per), off = (int)(local - (int64_t)item * per);
        const int take = (int)min((int64_t)(per - off), u1 - u);
        const int i0 = max(off - kSetup, 0), i1 = off + take - kSetup;  // blocks [i0, i1) of the item
        const int slot = u == u0 ? 0 : 1;  // a part is the share's first item or its last
        u += take;
        if (i1 <= i0) continue;
        const bool whole = i0 == 0 && i1 == w.nb;
        const int head = item / w.blocks, row0 = (item - head * w.blocks) * kCols;
        const int first_tok = (w.b0 + i0) * 16;
        // blocks of this part; a sequence of length 0 has one without tokens
        const int nblk = first_tok < w.length ? i1 - i0 : 0;

        // The page of block i of this part; negative: none that is in the cache.
        const int pp = a.page_size >> 4;
        auto page_of = [&](int i, int &blk) {
            blk = w.b0 + i0 + i;
            const int pg = blk / pp, page = __ldg(a.batch.table + (int64_t)b * a.batch.max_pages + pg);
            blk -= pg * pp;
            return page < a.pages ? page : -1;
        };
        // Row numbers / 16 in the cache of the next 32 blocks, one a lane.  Blocks
        // without a page stand at row 0; where there are any (true), all_vis becomes
        // INT_MIN: every step from then on is masked.
        uint32_t rows16 = 0;
        auto look_up = [&](int n0) {
            rows16 = 0;
            bool none = false;
            if (n0 + lane < nblk) {
                int blk;
                const int page = page_of(n0 + lane, blk);
                none = page < 0;
                if (none)
                    index_error();
                else
                    rows16 = (uint32_t)(((int64_t)page * a.kv_heads + head) * pp + blk);
            }
            return __any_sync(0xffffffffu, none) != 0;
        };
        auto load = [&](int i, int at) {  // block i, staged at byte `at` of the ring
            if (i < nblk) {
                const uint32_t r16 = __shfl_sync(0xffffffffu, rows16, i & 31);
                const uint32_t dst = ring_u + at;
#pragma unroll
                for (int j = 0; j < HD / 64; ++j) {
                    cp16(dst + to_codes + j * (32 / CH * kPitch), k_lane + (size_t)r16 * (16 * HD / 2) + j * 512);
                    cp16(dst + to_codes + j * (32 / CH * kPitch) + kCodes,
                         v_lane + (size_t)r16 * (16 * HD / 2) + j * 512);
                }
                if (lane < 4 * NG) cp16(dst + 2 * kCodes + lane * 16, sc_lane + (size_t)r16 * kScales);
            }
        };
        const bool holes = look_up(0);
        __syncwarp();  // the ring's last reads (of the item before) are done
#pragma unroll
        for (int i = 0; i < kStages; ++i) {
            load(i, i * kStage);
            if ((i + 1) % H == 0) cp_commit();
        }

        // ---- queries: column n = 8 j + g of this lane as B fragments
        uint32_t qf[NT][CH][4];
        float f[NT][2];            // factor of columns 8 j + 2 t4 and + 1
        int pos[NT][2];            // their positions
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int n = row0 + 8 * j + g;
            const bool in = n < w.rows;
            const int tk = in ? n / a.ratio : 0;
            const T *src = static_cast<const T *>(a.q) + (int64_t)(w.first + tk) * a.q_ts +
                           (int64_t)(head * a.ratio + (in ? n - tk * a.ratio : 0)) * a.q_hs;
            float top = 0.0f, v[8];
            if (!std::is_same<T, __half>::value) {
                if (in) {
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        load_q8<T>(src + 32 * c + 8 * t4, a.vec, v);
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            }
            float down;  // q * up in fp16, scores * down
            float up = fp16_power<T>(top, down);
            if (a.f < 0.0f) up = -up;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (in) load_q8<T>(src + 32 * c + 8 * t4, a.vec, v);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    qf[j][c][e] = in ? as_u32(__floats2half2_rn(v[e] * up, v[e + 4] * up)) : 0u;
            }
            const float fn = fmaxf(fabsf(a.f) * down, 1e-30f);  // not 0: masked scores are -inf before the product
            f[j][0] = __shfl_sync(0xffffffffu, fn, 8 * t4);
            f[j][1] = __shfl_sync(0xffffffffu, fn, 8 * t4 + 4);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = row0 + 8 * j + 2 * t4 + e;
                pos[j][e] = w.base + (col < w.rows ? col / a.ratio : w.count - 1);
            }
        }
        // tokens that every column of the item sees
        int all_vis = w.length, all_low = 0;
        if (a.causal) all_vis = w.base + row0 / a.ratio + 1;
        if (a.window > 0) {
            const int last = min(row0 + kCols, w.rows) - 1;
            all_low = (int)max((int64_t)w.base + last / a.ratio + 1 - a.window, (int64_t)0);
        }
        if (holes) all_vis = INT_MIN;

        float o[NT][HD / 16][4], m[NT][2], l[NT][2], most[NT][2];  // most: the score at which m is raised
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][i][e] = 0.0f;
            m[j][0] = m[j][1] = kNone;
            most[j][0] = most[j][1] = -INFINITY;
            l[j][0] = l[j][1] = 0.0f;
        }

        bool huge = false;  // a maximum of this lane's columns passed kHuge
        int at = 0;         // byte of the step in the ring
        for (int i = 0; i < nblk; i += H) {
            cp_wait<kSteps - 1>();
            __syncwarp();
            const int tok = first_tok + i * 16;

            // ---- scores of tokens g and g + 8 of the blocks
            float s[H][NT][4];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const unsigned char *st = ring + at + h * kStage;
                const uint32_t su = ring_u + at + h * kStage;
                uint32_t kw[2][CH];  // words t4 of each chunk of rows g, g + 8
                if (CH == 4) {
                    // matrix i of the four: chunk i of rows 0..7
                    const uint32_t ad = su + (lane & 7) * kPitch + (lane >> 3) * 16;
                    uint32_t r[4];
                    ldmatrix4(r, ad);
#pragma unroll
                    for (int c = 0; c < CH; ++c) kw[0][c] = r[c & 3];
                    ldmatrix4(r, ad + 8 * kPitch);
#pragma unroll
                    for (int c = 0; c < CH; ++c) kw[1][c] = r[c & 3];
                } else {
                    // chunks 0, 1 of rows 0..7, then of rows 8..15
                    uint32_t r[4];
                    ldmatrix4(r, su + ((lane & 7) + (lane >> 4) * 8) * kPitch + ((lane >> 3) & 1) * 16);
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        kw[0][c] = r[c & 1];
                        kw[1][c] = r[2 + (c & 1)];
                    }
                }
                alignas(8) __half ks[2][NG];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const unsigned char *p = st + 2 * kCodes + (g + 8 * x) * NG * 2;
                    if (NG == 4)
                        *reinterpret_cast<uint2 *>(ks[x]) = *reinterpret_cast<const uint2 *>(p);
                    else if (NG == 2)
                        *reinterpret_cast<uint32_t *>(ks[x]) = *reinterpret_cast<const uint32_t *>(p);
                    else
                        ks[x][0] = *reinterpret_cast<const __half *>(p);
                }
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    float acc[NT][4];
#pragma unroll
                    for (int cc = 0; cc < GS / 32; ++cc) {
                        const int c = G * (GS / 32) + cc;
                        __half2 x0[4], x1[4];
                        unpack_int(kw[0][c], x0);
                        unpack_int(kw[1][c], x1);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            if (cc == 0)
                                mma16816_first(acc[j], as_u32(x0[0]), as_u32(x1[0]), as_u32(x0[1]), as_u32(x1[1]),
                                               qf[j][c][0], qf[j][c][1]);
                            else
                                mma16816(acc[j], as_u32(x0[0]), as_u32(x1[0]), as_u32(x0[1]), as_u32(x1[1]),
                                         qf[j][c][0], qf[j][c][1]);
                            mma16816(acc[j], as_u32(x0[2]), as_u32(x1[2]), as_u32(x0[3]), as_u32(x1[3]), qf[j][c][2],
                                     qf[j][c][3]);
                        }
                    }
                    const float s0 = __half2float(ks[0][G]), s1 = __half2float(ks[1][G]);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float sc = e < 2 ? s0 : s1;
                            s[h][j][e] = G == 0 ? sc * acc[j][e] : fmaf(sc, acc[j][e], s[h][j][e]);
                        }
                }
            }

            // ---- weights p = 2^(s f - m)
            // some column misses some token of the blocks, or a block is not there
            const bool edge = tok + 16 * H > all_vis || tok < all_low || i + H > nblk;
            bool lost[H] = {};  // block i + h is not there
            if (edge) {
                const int64_t window = a.window > 0 ? a.window : INT32_MAX;
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    int blk;
                    lost[h] = i + h >= nblk;
                    if (all_vis == INT_MIN && !lost[h]) lost[h] = page_of(i + h, blk) < 0;
                }
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int tk = tok + 16 * h + g + (e >> 1) * 8, p = pos[j][e & 1];
                            const int vis = a.causal ? p + 1 : w.length;
                            if (tk >= vis || tk <= p - window || lost[h]) s[h][j][e] = -INFINITY;
                        }
            }
            bool raise = false;
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) raise |= s[h][j][e] > most[j][e & 1];
            if (__any_sync(0xffffffffu, raise)) {
                huge = false;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(s[0][j][e], s[0][j][e + 2]);
                        if (H == 2) mx = fmaxf(mx, fmaxf(s[H - 1][j][e], s[H - 1][j][e + 2]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float mn = fmaxf(m[j][e], __fmul_rn(mx, f[j][e]) - kLift);
                        const float corr = ex2(m[j][e] - mn);
                        m[j][e] = mn;
                        // (kNone passes kHuge too)
                        most[j][e] = fabsf(mn) > kHuge ? -INFINITY : __fdividef(mn + kRaise, f[j][e]);
                        huge |= fabsf(mn) > kHuge;
                        l[j][e] *= corr;
#pragma unroll
                        for (int i2 = 0; i2 < HD / 16; ++i2) {
                            o[j][i2][e] *= corr;
                            o[j][i2][e + 2] *= corr;
                        }
                    }
                if (huge) {
                    // (a column's lanes agree; from now on every step comes here)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        most[j][0] = most[j][1] = -INFINITY;
#pragma unroll
                        for (int h = 0; h < H; ++h)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[h][j][e] = __fmul_rn(s[h][j][e], f[j][e & 1]);
                    }
                }
            }
            uint32_t pf[H][NT][2];
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[e] = ex2(fmaf(s[h][j][e], huge ? 1.0f : f[j][e & 1], -m[j][e & 1]));
                        l[j][e & 1] += p[e];
                    }
                    pf[h][j][0] = transpose8x8(as_u32(__floats2half2_rn(p[0], p[1])));
                    pf[h][j][1] = transpose8x8(as_u32(__floats2half2_rn(p[2], p[3])));
                }

            // ---- o += V^T p: rows d = HD/8 g + ..., tokens 2 t4, +1, +8, +9
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const unsigned char *vc = ring + at + h * kStage + kCodes;
                const __half *vsc = reinterpret_cast<const __half *>(vc + kCodes + kScales);
                constexpr int W = HD / 64;  // words a lane takes of a token
                const int G = NG == 1 ? 0 : (HD / 8 * g) / GS;
                uint32_t vw[4][W];
                __half sc[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = 2 * t4 + (k & 1) + (k >> 1) * 8;
                    const uint32_t *src = reinterpret_cast<const uint32_t *>(vc + r * kPitch + g * (HD / 16));
                    if (W == 2) {
                        const uint2 two = *reinterpret_cast<const uint2 *>(src);
                        vw[k][0] = two.x;
                        vw[k][W - 1] = two.y;
                    } else {
                        vw[k][0] = src[0];
                    }
                    sc[k] = vsc[r * NG + G];
                }
                if (edge) {
                    // tokens that no row sees are whatever the page holds: no NaN from there
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int tk = tok + 16 * h + 2 * t4 + (k & 1) + (k >> 1) * 8;
                        if (tk >= w.length || tk < w.floor || lost[h]) sc[k] = __ushort_as_half(0);
                    }
                }
                const __half2 sa = __halves2half2(sc[0], sc[1]), sb = __halves2half2(sc[2], sc[3]);
#pragma unroll
                for (int x = 0; x < W; ++x) {
#pragma unroll
                    for (int hw = 0; hw < 2; ++hw) {  // codes 0..3, then 4..7 of the word
                        const uint32_t sel = hw ? 0x7632u : 0x5410u;
                        __half2 va[4], vb[4];
                        unpack_int(__byte_perm(vw[0][x], vw[1][x], sel), va);
                        unpack_int(__byte_perm(vw[2][x], vw[3][x], sel), vb);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            va[k] = __hmul2(va[k], sa);
                            vb[k] = __hmul2(vb[k], sb);
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int j = 0; j < NT; ++j)
                                mma16816(o[j][4 * x + 2 * hw + k], as_u32(va[2 * k]), as_u32(va[2 * k + 1]),
                                         as_u32(vb[2 * k]), as_u32(vb[2 * k + 1]), pf[h][j][0], pf[h][j][1]);
                    }
                }
            }
            __syncwarp();
            // later blocks take the place of these
            if (((i + kStages) & 31) == 0 && look_up(i + kStages)) all_vis = INT_MIN;
#pragma unroll
            for (int h = 0; h < H; ++h) load(i + kStages + h, at + h * kStage);
            cp_commit();
            at = at + H * kStage < kStages * kStage ? at + H * kStage : 0;
        }
        cp_wait<0>();

#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 4);
                l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 8);
                l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 16);
            }
        if (whole) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        write_slice<T, HD>(a, w, head, row0 + 8 * j + 2 * t4 + e, HD / 8 * g + 2 * i, o[j][i][e],
                                           o[j][i][e + 2], m[j][e], l[j][e]);
        } else {
            float *part = a.parts + (me * 2 + slot) * S::kPart;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (row0 + 8 * j + 2 * t4 < w.rows) {
                    if (g == 0) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            part[8 * j + 2 * t4 + e] = m[j][e];
                            part[kCols + 8 * j + 2 * t4 + e] = l[j][e];
                        }
                    }
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i)
                        reinterpret_cast<float4 *>(part + 2 * kCols)[(j * (HD / 16) + i) * 32 + lane] =
                            make_float4(o[j][i][0], o[j][i][1], o[j][i][2], o[j][i][3]);
                }
            }
        }
    }
    // Beside a prompt kernel, this one begins while that still runs (they
    // depend on nothing of each other), and must not be complete before it.
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Adds the parts of the items that more than one warp worked on, in order.  A
// CTA of eight warps an item; a slice is the float4 a lane holds of one
// product tile.  SPLIT: a CTA per slice, whose warps share the parts (many
// parts, few items); else a warp per slice.
template <typename T, int HD, int NT, bool SPLIT>
__global__ void __launch_bounds__(256) join_kernel(const Args a, int warps) {
    using S = Shape<HD, NT>;
    constexpr int kCols = S::kCols;
    // All but the parts is known before the streaming kernel is done.
    extern __shared__ __align__(16) unsigned char join_smem[];
    int64_t *prefix = reinterpret_cast<int64_t *>(join_smem);
    units_before<256>(a, kCols, prefix);
    const int b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const Work w = work_of(a, b, kCols);
    const int item = blockIdx.y;
    const bool there = item < w.blocks * a.kv_heads;
    const int64_t all = max(prefix[a.batch.sequences], (int64_t)1), shares = shares_of(all, warps);
    const int64_t s = prefix[b] + (int64_t)item * (w.nb + kSetup), e = s + w.nb + kSetup;
    // the warp that worked on unit u: the last i with i all / shares <= u
    const int64_t c0 = quotient((s + kSetup + 1) * shares - 1, all), c1 = quotient(e * shares - 1, all);
    // (every warp between them has units, as shares <= all; only the first may start before the item)
    const bool late = quotient(c0 * all, shares) >= s;
    // (also by a CTA that has nothing to do: this kernel is not complete before the other)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (w.out) {
        // (here, as the streaming kernel's code begins cold at every launch: clearing
        // them there cost one request of 1000 tokens 0.3 us of 10.75)
        index_error();
        const int64_t row0 = (int64_t)w.first * a.q_heads, row1 = row0 + (int64_t)w.count * a.q_heads;
        int64_t row = row0 + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 8 + warp;
        for (; row < row1; row += (int64_t)gridDim.x * gridDim.y * 8) {
            for (int i = lane; i < HD; i += 32) put(static_cast<T *>(a.out) + row * HD + i, 0.0f);
            if (lane == 0 && a.log_sum != nullptr) a.log_sum[row] = -INFINITY;
        }
        return;
    }
    if (!there || c0 == c1) return;
    const int head = item / w.blocks, row0 = (item - head * w.blocks) * kCols;
    const float *first = a.parts + (c0 * 2 + (late ? 0 : 1)) * S::kPart;
    const float *rest = a.parts + c0 * 2 * S::kPart;  // part n > 0: rest + n * 2 * kPart
    const int parts = (int)(c1 - c0) + 1;
    __shared__ float4 so[8][32];
    __shared__ float sm[8][kCols], sl[8][kCols];
    for (int sl_i = SPLIT ? (int)blockIdx.x : warp; sl_i < S::kSlices; sl_i += SPLIT ? S::kSlices : 8) {
        const int j = sl_i / (HD / 16), i = sl_i % (HD / 16), col = 8 * j + 2 * t4;
        const bool in = row0 + col < w.rows;
        // of the lane's two columns, over the parts so far
        float m[2] = {kNone, kNone}, l[2] = {0.0f, 0.0f};
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (in) {
            constexpr int U = 8;  // parts in flight
            for (int n0 = SPLIT ? warp : 0; n0 < parts; n0 += SPLIT ? 8 * U : U) {
                float4 v[U];
                float pm[U][2], pl[U][2], mn[2] = {m[0], m[1]};
#pragma unroll
                for (int x = 0; x < U; ++x) {
                    const int n = n0 + (SPLIT ? 8 * x : x);
                    const float *p = n == 0 ? first : rest + (int64_t)n * 2 * S::kPart;
                    v[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    pm[x][0] = pm[x][1] = -INFINITY;
                    pl[x][0] = pl[x][1] = 0.0f;
                    if (n < parts) {
                        v[x] = reinterpret_cast<const float4 *>(p + 2 * kCols)[sl_i * 32 + lane];
                        pm[x][0] = p[col], pm[x][1] = p[col + 1];
                        pl[x][0] = p[kCols + col], pl[x][1] = p[kCols + col + 1];
                    }
                }
#pragma unroll
                for (int x = 0; x < U; ++x) mn[0] = fmaxf(mn[0], pm[x][0]), mn[1] = fmaxf(mn[1], pm[x][1]);
                const float k0 = ex2(m[0] - mn[0]), k1 = ex2(m[1] - mn[1]);
                m[0] = mn[0], m[1] = mn[1];
                l[0] *= k0, o.x *= k0, o.z *= k0;
                l[1] *= k1, o.y *= k1, o.w *= k1;
#pragma unroll
                for (int x = 0; x < U; ++x) {
                    const float c = ex2(pm[x][0] - m[0]), d = ex2(pm[x][1] - m[1]);
                    l[0] = fmaf(c, pl[x][0], l[0]);
                    l[1] = fmaf(d, pl[x][1], l[1]);
                    o.x = fmaf(c, v[x].x, o.x), o.z = fmaf(c, v[x].z, o.z);
                    o.y = fmaf(d, v[x].y, o.y), o.w = fmaf(d, v[x].w, o.w);
                }
            }
        }
        if (SPLIT) {
            so[warp][lane] = o;
            if (g == 0) {
#pragma unroll
                for (int x = 0; x < 2; ++x) sm[warp][col + x] = m[x], sl[warp][col + x] = l[x];
            }
            __syncthreads();
            if (warp != 0) return;
            float mn[2] = {m[0], m[1]};
#pragma unroll
            for (int k = 1; k < 8; ++k) mn[0] = fmaxf(mn[0], sm[k][col]), mn[1] = fmaxf(mn[1], sm[k][col + 1]);
            l[0] = l[1] = 0.0f;
            o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float c = ex2(sm[k][col] - mn[0]), d = ex2(sm[k][col + 1] - mn[1]);
                const float4 v = so[k][lane];
                l[0] = fmaf(c, sl[k][col], l[0]);
                l[1] = fmaf(d, sl[k][col + 1], l[1]);
                o.x = fmaf(c, v.x, o.x), o.z = fmaf(c, v.z, o.z);
                o.y = fmaf(d, v.y, o.y), o.w = fmaf(d, v.w, o.w);
            }
            m[0] = mn[0], m[1] = mn[1];
        }
        write_slice<T, HD>(a, w, head, row0 + col, HD / 8 * g + 2 * i, o.x, o.z, m[0], l[0]);
        write_slice<T, HD>(a, w, head, row0 + col + 1, HD / 8 * g + 2 * i, o.y, o.w, m[1], l[1]);
    }
}

// CTAs of the streaming kernel: what fits on the GPU at once.
template <int HD, int NT>
int share_of() { return sm_count() * kCtas<HD, NT>; }

int share_of(const oq_kv4_cache *c, int nt) {
    if (c->head_dim == 64) return nt == 1 ? share_of<64, 1>() : share_of<64, 2>();
    return nt == 1 ? share_of<128, 1>() : share_of<128, 2>();
}

template <int HD, int GS>
constexpr size_t ring_bytes() {
    return (size_t)kWarps * kStages * (2 * 16 * (HD / 2 + 16) + 2 * 16 * (HD / GS) * 2);
}

// Sequences of up to this many query rows a key head are streamed (in blocks of
// 16 rows, each of which reads the cache again, from L2), the others go to the
// prompt kernel, whose tiles have 128 rows.  Single tokens are always streamed.
// Measured, streamed / prompt kernel: head_dim 64, 37 rows over 23 x 11139
// tokens 160 / 185 us, 48 rows over 34 x 8902..17804 tokens 50 / 62 us; head_dim
// 128, 40 rows over 16 x 8000 tokens 142 / 112 us, 64 rows 186 / 113 us (32 rows,
// streamed, 99 us).
int few_rows(const oq_kv4_cache *c, int q_heads) {
    const int ratio = q_heads / c->kv_heads, few = c->head_dim == 64 ? 64 : 32;
    return ratio > few ? ratio : few;
}

int columns_of(const oq_kv4_cache *c, const oq_kv4_batch *b, int q_heads) {
    return (int64_t)b->max_tokens * (q_heads / c->kv_heads) <= 8 ? 1 : 2;
}

// Items of a sequence that the streaming kernel may have to join: a block of
// the joining kernel's grid in y.
int64_t join_items(int kv_heads, int ratio, int few, const oq_kv4_batch *b, int nt) {
    const int64_t most = (int64_t)b->max_tokens * ratio;
    return cdiv(most < few ? most : few, 8 * nt) * kv_heads;
}

template <typename T, int HD, int GS, int NT>
int stream_launch(Args &a, const oq_kv4_batch *batch, bool beside, cudaStream_t st) {
    const int share = share_of<HD, NT>();
    auto kern = stream_kernel<T, HD, GS, NT>;
    const size_t smem = ring_bytes<HD, GS>() + (batch->sequences + 1) * 8;  // the prefix follows the rings
    if (int rc = allow_dynamic_smem(reinterpret_cast<const void *>(kern), smem)) return rc;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(share);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = beside ? 1 : 0;
    cudaError_t err = cudaLaunchKernelEx(&cfg, kern, (const Args)a);
    if (err != cudaSuccess) {
        set_error("kv4_attention: launch failed: %s", cudaGetErrorString(err));
        return OQ_ERR_CUDA;
    }

    const int64_t items = join_items(a.kv_heads, a.ratio, a.few, batch, NT);
    const int warps = share * kWarps;
    const bool split = warps > 16 * items * batch->sequences;
    cfg.gridDim = dim3(split ? Shape<HD, NT>::kSlices : 1, (unsigned)items, batch->sequences);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = (batch->sequences + 1) * 8;
    cfg.numAttrs = 1;
    err = split ? cudaLaunchKernelEx(&cfg, join_kernel<T, HD, NT, true>, a, warps)
                            : cudaLaunchKernelEx(&cfg, join_kernel<T, HD, NT, false>, a, warps);
    if (err != cudaSuccess) {
        set_error("kv4_attention (join): launch failed: %s", cudaGetErrorString(err));
        return OQ_ERR_CUDA;
    }
    return OQ_OK;
}

template <typename T, int HD, int GS>
int stream_columns(Args &a, const oq_kv4_batch *batch, int nt, bool beside, cudaStream_t st) {
    return nt == 1 ? stream_launch<T, HD, GS, 1>(a, batch, beside, st)
                   : stream_launch<T, HD, GS, 2>(a, batch, beside, st);
}

template <typename T>
int attention_typed(Args &a, const oq_kv4_cache *c, const oq_kv4_batch *batch, int nt, bool beside,
                    cudaStream_t st) {
    if (c->head_dim == 64)
        return c->group_size == 32 ? stream_columns<T, 64, 32>(a, batch, nt, beside, st)
                                   : stream_columns<T, 64, 64>(a, batch, nt, beside, st);
    return c->group_size == 32   ? stream_columns<T, 128, 32>(a, batch, nt, beside, st)
           : c->group_size == 64 ? stream_columns<T, 128, 64>(a, batch, nt, beside, st)
                                 : stream_columns<T, 128, 128>(a, batch, nt, beside, st);
}

// Workspace of the streaming kernel.
int64_t stream_bytes(const oq_kv4_cache *c, const oq_kv4_batch *b, int q_heads) {
    const int nt = columns_of(c, b, q_heads);
    const int64_t warps = (int64_t)share_of(c, nt) * kWarps;
    return warps * 2 * (16 * nt + nt * c->head_dim * 8) * 4;
}

// Items of the prompt kernel at most: the sum over sequences of ceil(rows / kPromptRows).
int64_t prompt_items(const oq_kv4_cache *c, const oq_kv4_batch *b, int q_heads, int64_t tokens) {
    const int64_t ratio = q_heads / c->kv_heads, most = cdiv(b->max_tokens * ratio, kPromptRows) * b->sequences;
    const int64_t bound = cdiv(tokens * ratio, kPromptRows) + b->sequences - 1;
    return (bound < most ? bound : most) * c->kv_heads;
}

int check_heads(const oq_kv4_cache *c, int q_heads) {
    OQ_REQUIRE(q_heads >= 1 && q_heads % c->kv_heads == 0, "kv4_attention: q_heads must be a multiple of kv_heads");
    return OQ_OK;
}

}  // namespace
}  // namespace kv4
}  // namespace oq

using namespace oq;
using namespace oq::kv4;

extern "C" int64_t oq_kv4_attention_workspace_bytes(const oq_kv4_cache *cache, const oq_kv4_batch *batch, int q_heads,
                                                    int64_t tokens) {
    clear_error();
    if (check_cache(cache) || check_batch(batch, tokens) || check_heads(cache, q_heads)) return 0;
    const int64_t ratio = q_heads / cache->kv_heads;
    int64_t n = stream_bytes(cache, batch, q_heads);
    if (batch->max_tokens * ratio > few_rows(cache, q_heads)) {
        const int64_t items = prompt_items(cache, batch, q_heads, tokens);
        n += prompt_part_bytes(cache, items, prompt_cuts(cache, batch, items));
    }
    return n;
}

extern "C" int oq_kv4_attention(const oq_kv4_cache *cache, const oq_kv4_batch *batch, const void *q, int dtype,
                                int q_heads, int64_t q_token_stride, int64_t q_head_stride, void *out, float *log_sum,
                                int64_t tokens, float scale, int64_t window, int flags, void *workspace,
                                size_t ws_bytes, oq_stream_t stream) {
    clear_error();
    OQ_REQUIRE(dtype == OQ_F16 || dtype == OQ_BF16, "kv4_attention: q must be fp16 or bf16");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(batch, tokens)) return rc;
    if (int rc = check_heads(cache, q_heads)) return rc;
    OQ_REQUIRE(q && out && workspace, "null pointer argument");
    OQ_REQUIRE(aligned(out, 16) && aligned(workspace, 16), "kv4_attention: out and workspace must be 16-byte aligned");
    OQ_REQUIRE(window >= 0, "kv4_attention: window must not be negative");
    OQ_REQUIRE((flags & ~OQ_KV4_NOT_CAUSAL) == 0, "kv4_attention: unknown flags");
    const float f = scale * 1.4426950408889634f;
    OQ_REQUIRE(f - f == 0.0f, "kv4_attention: scale must be finite, times log2 e too");
    OQ_REQUIRE((int64_t)ws_bytes >= oq_kv4_attention_workspace_bytes(cache, batch, q_heads, tokens),
               "kv4_attention: workspace too small");
    Args a = {};
    a.k_codes = cache->k_codes;
    a.v_codes = cache->v_codes;
    a.k_scales = static_cast<const __half *>(cache->k_scales);
    a.v_scales = static_cast<const __half *>(cache->v_scales);
    a.pages = cache->pages;
    a.page_size = cache->page_size;
    a.kv_heads = cache->kv_heads;
    a.batch = device_batch(batch);
    a.q = q;
    a.q_ts = q_token_stride;
    a.q_hs = q_head_stride;
    a.out = out;
    a.log_sum = log_sum;
    a.tokens = tokens;
    a.max_tokens = batch->max_tokens;
    a.q_heads = q_heads;
    a.ratio = q_heads / cache->kv_heads;
    a.f = f;
    a.window = window < INT32_MAX ? window : 0;  // positions are below 2^31: no limit
    a.causal = (flags & OQ_KV4_NOT_CAUSAL) ? 0 : 1;
    a.parts = static_cast<float *>(workspace);
    a.vec = aligned(q, 16) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
    const int nt = columns_of(cache, batch, q_heads);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t most = (int64_t)batch->max_tokens * a.ratio;  // rows a sequence and key head
    a.few = few_rows(cache, q_heads);
    // (before any launch: a refused call does nothing)
    OQ_REQUIRE(join_items(a.kv_heads, a.ratio, a.few, batch, nt) <= 65535, "kv4_attention: too many key heads");
    const bool beside = most > a.few;
    if (beside) {
        AttnArgs p = a;
        p.parts = reinterpret_cast<float *>(static_cast<char *>(workspace) + stream_bytes(cache, batch, q_heads));
        const int64_t items = prompt_items(cache, batch, q_heads, tokens);
        if (int rc = prompt_attention(p, dtype, cache, items, prompt_cuts(cache, batch, items), st)) return rc;
    }
    return dtype == OQ_F16 ? attention_typed<__half>(a, cache, batch, nt, beside, st)
                           : attention_typed<__nv_bfloat16>(a, cache, batch, nt, beside, st);
}
