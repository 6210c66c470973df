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
#include "oq_kv4_attention.cuh"

namespace oq {
namespace kv4 {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 16 * kWarps;  // cached tokens of one round of a CTA
constexpr int kStages = 4;          // 16-token stages a warp has in flight or in use

using Args = AttnArgs;

// Columns (query rows) of a partial, and its floats: m[cols], l[cols], o[cols][HD].
template <int HD, int NT>
struct Shape {
    static constexpr int kCols = 8 * NT;
    static constexpr int kPart = kCols * (HD + 2);
    static constexpr int kPitch = HD / 2 + 16;  // bytes of a staged row: 16-byte steps over all banks
};

// Work of sequence b: `tiles` rounds per item, an item per key head and per
// block of kCols query rows.
struct Work {
    int first, count, rows, length;
    int64_t floor;  // first cached token any row sees
    int64_t lo;     // the same down to a tile
    int tiles, blocks;
};

__device__ __forceinline__ Work work_of(const Args &a, int b, int cols) {
    Work w;
    tokens_of(a.batch, b, a.tokens, w.first, w.count);
    w.length = length_of(a.batch, b, a.page_size);
    w.rows = w.count * a.ratio;
    w.blocks = w.rows > a.few ? 0 : (w.rows + cols - 1) / cols;
    w.floor = 0;
    if (a.window > 0) w.floor = max((int64_t)w.length - w.count + 1 - a.window, (int64_t)0);
    w.lo = w.floor / kTile * kTile;
    const int64_t n = ((int64_t)w.length - w.lo + kTile - 1) / kTile;
    w.tiles = n > 1 ? (int)n : 1;
    return w;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// One CTA = four warps over an equal share of all rounds (64 tokens of one
// item), so that ragged lengths load every SM alike: a share begins and ends
// inside an item, whose parts the joining kernel adds in a fixed order.  A
// warp streams its own 16 tokens of each round through a ring of cp.async
// stages; the rows are staged 16 bytes longer than they are, which makes both
// the ldmatrix of the keys and the 4- or 8-byte reads of the values free of
// bank conflicts.
template <typename T, int HD, int GS, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 4 : 3) stream_kernel(const Args a) {
    using S = Shape<HD, NT>;
    constexpr int kCols = S::kCols, kPitch = S::kPitch;
    constexpr int NG = HD / GS;             // groups a row
    constexpr int CH = HD / 32;             // 16-byte chunks a row
    constexpr int kCodes = 16 * kPitch;     // staged codes of 16 tokens
    constexpr int kScales = 16 * NG * 2;
    constexpr int kStage = 2 * kCodes + 2 * kScales;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    unsigned char *ring = smem + warp * kStages * kStage;
    int64_t *prefix = reinterpret_cast<int64_t *>(smem + kWarps * kStages * kStage);

    // ---- units before each sequence (exclusive prefix in shared memory)
    {
        __shared__ int64_t warp_sum[kWarps];
        int64_t base = 0;
        for (int b0 = 0; b0 < a.batch.sequences; b0 += kWarps * 32) {
            const int b = b0 + tid;
            int64_t n = 0;
            if (b < a.batch.sequences) {
                const Work w = work_of(a, b, kCols);
                n = (int64_t)w.tiles * w.blocks * a.kv_heads;
            }
            int64_t inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            if (lane == 31) warp_sum[warp] = inc;
            __syncthreads();
            int64_t before = base, all = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) before += warp_sum[w];
                all += warp_sum[w];
            }
            if (b < a.batch.sequences) prefix[b] = before + inc - n;
            base += all;
            __syncthreads();
        }
        if (tid == 0) prefix[a.batch.sequences] = base;
        __syncthreads();
        if (blockIdx.x == 0)
            for (int b = tid; b <= a.batch.sequences; b += kWarps * 32) a.prefix[b] = prefix[b];
    }
    const int64_t all = prefix[a.batch.sequences];
    const int64_t u0 = (int64_t)blockIdx.x * all / gridDim.x, u1 = ((int64_t)blockIdx.x + 1) * all / gridDim.x;

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
        const int item = (int)(local / w.tiles), tile0 = (int)(local - (int64_t)item * w.tiles);
        const int tile1 = (int)min((int64_t)w.tiles, tile0 + (u1 - u));
        const int head = item / w.blocks, row0 = (item - head * w.blocks) * kCols;
        const bool whole = tile0 == 0 && tile1 == w.tiles;
        const int slot = u == u0 ? 0 : 1;  // a part is the share's first item or its last
        u += tile1 - tile0;

        // ---- this warp's 16-token blocks: tokens tok0 + i * kTile, i < nblk
        const int64_t tok0 = w.lo + (int64_t)tile0 * kTile + warp * 16;
        int nblk = tile1 - tile0;
        {
            const int64_t left = (int64_t)w.length - tok0;  // tokens from tok0 on
            const int64_t most = left > 0 ? (left + kTile - 1) / kTile : 0;
            if (most < nblk) nblk = (int)most;
        }

        // Row numbers / 16 in the cache of the next 32 blocks, one a lane.
        uint32_t rows16 = 0;
        auto look_up = [&](int i0) {
            const int i = i0 + lane;
            rows16 = 0;
            // blocks below every window are staged (row 0 of the cache) but not looked up:
            // their pages may be gone
            if (i < nblk && tok0 + (int64_t)i * kTile + 16 > w.floor) {
                const int64_t blk = (tok0 + (int64_t)i * kTile) >> 4;
                const int per = a.page_size >> 4;
                const int pg = (int)(blk / per);
                const int page = __ldg(a.batch.table + (int64_t)b * a.batch.max_pages + pg);
                if (page < 0 || page >= a.pages)
                    index_error();
                else
                    rows16 = (uint32_t)(((int64_t)page * a.kv_heads + head) * per + (blk - (int64_t)pg * per));
            }
        };
        auto load = [&](int i) {
            if (i < nblk) {
                const uint32_t r16 = __shfl_sync(0xffffffffu, rows16, i & 31);
                unsigned char *st = ring + (i % kStages) * kStage;
                const uint32_t dst = smem_u32(st);
                const uint8_t *ks = a.k_codes + (size_t)r16 * (16 * HD / 2);
                const uint8_t *vs = a.v_codes + (size_t)r16 * (16 * HD / 2);
#pragma unroll
                for (int j = 0; j < HD / 64; ++j) {
                    const int ch = lane + 32 * j;
                    const uint32_t to = dst + (ch / CH) * kPitch + (ch % CH) * 16;
                    cp16(to, ks + ch * 16);
                    cp16(to + kCodes, vs + ch * 16);
                }
                if (lane < 2 * NG)
                    cp16(dst + 2 * kCodes + lane * 16,
                         reinterpret_cast<const unsigned char *>(a.k_scales) + (size_t)r16 * kScales + lane * 16);
                else if (lane < 4 * NG)
                    cp16(dst + 2 * kCodes + lane * 16, reinterpret_cast<const unsigned char *>(a.v_scales) +
                                                           (size_t)r16 * kScales + (lane - 2 * NG) * 16);
            }
            cp_commit();
        };
        look_up(0);
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) load(i);

        // ---- queries: column n = 8 j + g of this lane as B fragments
        uint32_t qf[NT][CH][4];
        float f[NT][2];              // factor of columns 8 j + 2 t4 and + 1
        int64_t vis[NT][2], low[NT][2];  // their visible tokens [low, vis)
        int64_t all_vis = w.length, all_low = 0;  // visible to every column
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int n = row0 + 8 * j + g;
            const bool in = n < w.rows;
            const int tk = in ? n / a.ratio : 0;
            const T *src = static_cast<const T *>(a.q) + (int64_t)(w.first + tk) * a.q_ts +
                           (int64_t)(head * a.ratio + (in ? n - tk * a.ratio : 0)) * a.q_hs;
            float top = 0.0f;
            float v[CH][8];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (in) load_q8<T>(src + 32 * c + 8 * t4, a.vec, v[c]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (!in) v[c][e] = 0.0f;
                    top = fmaxf(top, fabsf(v[c][e]));
                }
            }
            if (!std::is_same<T, __half>::value) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            }
            float down;  // q * up in fp16, scores * down
            const float up = fp16_power<T>(top, down);
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    qf[j][c][e] = as_u32(__floats2half2_rn(v[c][e] * up, v[c][e + 4] * up));
            const float fn = a.f * down;
            f[j][0] = __shfl_sync(0xffffffffu, fn, 8 * t4);
            f[j][1] = __shfl_sync(0xffffffffu, fn, 8 * t4 + 4);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = row0 + 8 * j + 2 * t4 + e;
                const int64_t p = (int64_t)w.length - w.count + (col < w.rows ? col / a.ratio : w.count - 1);
                vis[j][e] = a.causal ? p + 1 : w.length;
                low[j][e] = a.window > 0 ? p + 1 - a.window : 0;
            }
        }
        {
            const int64_t p0 = (int64_t)w.length - w.count + row0 / a.ratio;  // the first row's position
            if (a.causal) all_vis = p0 + 1;
            if (a.window > 0) {
                const int last = min(row0 + kCols, w.rows) - 1;
                all_low = (int64_t)w.length - w.count + last / a.ratio + 1 - a.window;
            }
        }

        float o[NT][HD / 16][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][i][e] = 0.0f;
            m[j][0] = m[j][1] = -1e30f;
            l[j][0] = l[j][1] = 0.0f;
        }

        for (int i = 0; i < nblk; ++i) {
            // stage i + kStages - 1 takes the place of stage i - 1, whose reads
            // ended before the warp's last __syncwarp
            if (((i + kStages - 1) & 31) == 0) look_up(i + kStages - 1);
            load(i + kStages - 1);
            cp_wait<kStages - 1>();
            __syncwarp();
            const unsigned char *st = ring + (i % kStages) * kStage;
            const uint32_t su = smem_u32(st);
            const int64_t tok = tok0 + (int64_t)i * kTile;

            // ---- scores of tokens g and g + 8
            float s[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
            {
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
                const __half *ksc = reinterpret_cast<const __half *>(st + 2 * kCodes);
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    float acc[NT][4];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
#pragma unroll
                    for (int cc = 0; cc < GS / 32; ++cc) {
                        const int c = G * (GS / 32) + cc;
                        __half2 x0[4], x1[4];
                        unpack_int(kw[0][c], x0);
                        unpack_int(kw[1][c], x1);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            mma16816(acc[j], as_u32(x0[0]), as_u32(x1[0]), as_u32(x0[1]), as_u32(x1[1]), qf[j][c][0],
                                     qf[j][c][1]);
                            mma16816(acc[j], as_u32(x0[2]), as_u32(x1[2]), as_u32(x0[3]), as_u32(x1[3]), qf[j][c][2],
                                     qf[j][c][3]);
                        }
                    }
                    const float s0 = __half2float(ksc[g * NG + G]), s1 = __half2float(ksc[(g + 8) * NG + G]);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        s[j][0] += s0 * acc[j][0];
                        s[j][1] += s0 * acc[j][1];
                        s[j][2] += s1 * acc[j][2];
                        s[j][3] += s1 * acc[j][3];
                    }
                }
            }

            // ---- weights p = 2^(s f - m)
            const bool edge = tok + 16 > all_vis || tok < all_low;  // warp-uniform: some column misses some token
            bool raise = false;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = s[j][e] * f[j][e & 1];
                    if (edge) {
                        const int64_t tk = tok + g + (e >> 1) * 8;
                        if (tk >= vis[j][e & 1] || tk < low[j][e & 1]) x = -INFINITY;
                    }
                    s[j][e] = x;
                    raise |= x > m[j][e & 1] + kRaise;
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(s[j][e], s[j][e + 2]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float mn = fmaxf(m[j][e], mx - kLift);
                        const float corr = ex2(m[j][e] - mn);
                        m[j][e] = mn;
                        l[j][e] *= corr;
#pragma unroll
                        for (int i2 = 0; i2 < HD / 16; ++i2) {
                            o[j][i2][e] *= corr;
                            o[j][i2][e + 2] *= corr;
                        }
                    }
            }
            uint32_t pf[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = ex2(s[j][e] - m[j][e & 1]);
                    l[j][e & 1] += p[e];
                }
                pf[j][0] = transpose8x8(as_u32(__floats2half2_rn(p[0], p[1])));
                pf[j][1] = transpose8x8(as_u32(__floats2half2_rn(p[2], p[3])));
            }

            // ---- o += V^T p: rows d = HD/8 g + ..., tokens 2 t4, +1, +8, +9
            {
                const unsigned char *vc = st + kCodes;
                const __half *vsc = reinterpret_cast<const __half *>(st + 2 * kCodes + kScales);
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
                    // tokens that no row sees are whatever the page holds: no NaN from there
                    if (edge && (tok + r >= w.length || tok + r < w.floor)) sc[k] = __ushort_as_half(0);
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
                                         as_u32(vb[2 * k]), as_u32(vb[2 * k + 1]), pf[j][0], pf[j][1]);
                    }
                }
            }
            __syncwarp();
        }
        cp_wait<0>();
        __syncthreads();

        // ---- join the four warps (the ring is free: every copy has landed)
        float *wm = reinterpret_cast<float *>(smem), *wl = wm + kWarps * kCols, *wo = wl + kWarps * kCols;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = l[j][e];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int col = 8 * j + 2 * t4 + e;
                if (g == 0) {
                    wm[warp * kCols + col] = m[j][e];
                    wl[warp * kCols + col] = x;
                }
                float *dst = wo + (size_t)(warp * kCols + col) * HD + HD / 8 * g;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i)
                    *reinterpret_cast<float2 *>(dst + 2 * i) = make_float2(o[j][i][e], o[j][i][e + 2]);
            }
        }
        __syncthreads();
        float *part = a.parts + ((int64_t)blockIdx.x * 2 + slot) * S::kPart;
        for (int x = tid; x < kCols * HD / 4; x += kWarps * 32) {
            const int col = x / (HD / 4), d = x % (HD / 4) * 4;
            float mx = wm[col];
#pragma unroll
            for (int k = 1; k < kWarps; ++k) mx = fmaxf(mx, wm[k * kCols + col]);
            float sum = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float c = ex2(wm[k * kCols + col] - mx);
                const float4 ov = *reinterpret_cast<const float4 *>(wo + (size_t)(k * kCols + col) * HD + d);
                sum += c * wl[k * kCols + col];
                v.x += c * ov.x, v.y += c * ov.y, v.z += c * ov.z, v.w += c * ov.w;
            }
            if (!whole) {
                if (d == 0) {
                    part[col] = mx;
                    part[kCols + col] = sum;
                }
                *reinterpret_cast<float4 *>(part + 2 * kCols + col * HD + d) = v;
            } else if (row0 + col < w.rows) {
                const int n = row0 + col, tk = n / a.ratio;
                const int64_t row = (int64_t)(w.first + tk) * a.q_heads + head * a.ratio + (n - tk * a.ratio);
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                T *dst = static_cast<T *>(a.out) + row * HD + d;
                put(dst, v.x * inv), put(dst + 1, v.y * inv), put(dst + 2, v.z * inv), put(dst + 3, v.w * inv);
                if (d == 0 && a.log_sum != nullptr)
                    a.log_sum[row] = sum == 0.0f ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
            }
        }
        __syncthreads();
    }
}

// Adds the parts of the items that more than one CTA worked on, in order.  A
// CTA of eight warps per item: with SPLIT each of its columns has a CTA of
// its own whose warps share the parts, else each warp takes whole columns.
template <typename T, int HD, int NT, bool SPLIT>
__global__ void __launch_bounds__(256) join_kernel(const Args a, int share) {
    using S = Shape<HD, NT>;
    constexpr int kCols = S::kCols, V = HD / 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Work w = work_of(a, b, kCols);
    const int item = blockIdx.y;
    if (item >= w.blocks * a.kv_heads) return;
    const int64_t all = a.prefix[a.batch.sequences], s = a.prefix[b] + (int64_t)item * w.tiles, e = s + w.tiles;
    // the CTA that worked on unit u: the last i with i all / share <= u
    const int64_t c0 = ((s + 1) * share - 1) / all, c1 = (e * share - 1) / all;
    if (c0 == c1) return;
    const int head = item / w.blocks, row0 = (item - head * w.blocks) * kCols;
    __shared__ float sm[8], sl[8], so[8][HD];
    for (int col = SPLIT ? (int)blockIdx.x : warp; col < kCols; col += SPLIT ? kCols : 8) {
        if (row0 + col >= w.rows) break;  // rows of a block are in order: the rest are past the end too
        float m = -1e30f, l = 0.0f, o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = 0.0f;
        for (int64_t c = c0 + (SPLIT ? warp : 0); c <= c1; c += SPLIT ? 8 : 1) {
            const int64_t from = c * all / share, to = (c + 1) * all / share;
            if (from == to) continue;  // a CTA without work
            const float *p = a.parts + (c * 2 + (from >= s ? 0 : 1)) * S::kPart;
            const float pm = p[col], pl = p[kCols + col];
            float pv[V];
#pragma unroll
            for (int i = 0; i < V; ++i) pv[i] = p[2 * kCols + col * HD + i * 32 + lane];
            const float mn = fmaxf(m, pm), x = ex2(m - mn), y = ex2(pm - mn);
            m = mn;
            l = l * x + pl * y;
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = o[i] * x + pv[i] * y;
        }
        if (SPLIT) {
            if (lane == 0) {
                sm[warp] = m;
                sl[warp] = l;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) so[warp][i * 32 + lane] = o[i];
            __syncthreads();
            if (warp != 0) return;
            for (int k = 1; k < 8; ++k) {
                const float mn = fmaxf(m, sm[k]), x = ex2(m - mn), y = ex2(sm[k] - mn);
                m = mn;
                l = l * x + sl[k] * y;
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = o[i] * x + so[k][i * 32 + lane] * y;
            }
        }
        const int n = row0 + col, tk = n / a.ratio;
        const int64_t row = (int64_t)(w.first + tk) * a.q_heads + head * a.ratio + (n - tk * a.ratio);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < V; ++i) put(static_cast<T *>(a.out) + row * HD + i * 32 + lane, o[i] * inv);
        if (lane == 0 && a.log_sum != nullptr)
            a.log_sum[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
}

// CTAs of the streaming kernel: what fits on the GPU at once.
template <int NT>
int share_of() { return sm_count() * (NT == 1 ? 4 : 3); }

template <int HD, int GS>
constexpr size_t ring_bytes() {
    return (size_t)kWarps * kStages * (2 * 16 * (HD / 2 + 16) + 2 * 16 * (HD / GS) * 2);
}

size_t header_bytes(const oq_kv4_batch *b) { return (size_t)cdiv((b->sequences + 1) * 8, 128) * 128; }

// Sequences of up to kFew query rows a key head are streamed, the others go to
// the prompt kernel.
constexpr int kFew = 32;

int columns_of(const oq_kv4_cache *c, const oq_kv4_batch *b, int q_heads) {
    return (int64_t)b->max_tokens * (q_heads / c->kv_heads) <= 8 ? 1 : 2;
}

template <typename T, int HD, int GS, int NT>
int stream_launch(Args &a, const oq_kv4_batch *batch, cudaStream_t st) {
    const int share = share_of<NT>();
    auto kern = stream_kernel<T, HD, GS, NT>;
    const size_t red = (size_t)kWarps * Shape<HD, NT>::kPart * 4;
    const size_t ring = ring_bytes<HD, GS>() > red ? ring_bytes<HD, GS>() : red;
    // the prefix follows the ring
    const size_t smem = ring_bytes<HD, GS>() + (batch->sequences + 1) * 8 > ring
                            ? ring_bytes<HD, GS>() + (batch->sequences + 1) * 8
                            : ring;
    static_assert(ring_bytes<HD, GS>() >= (size_t)kWarps * Shape<HD, NT>::kPart * 4, "the join fits the ring");
    if (int rc = allow_dynamic_smem(reinterpret_cast<const void *>(kern), smem)) return rc;
    kern<<<share, kWarps * 32, smem, st>>>(a);
    if (int rc = check_launch("kv4_attention")) return rc;

    const int64_t most = (int64_t)batch->max_tokens * a.ratio;
    const int64_t blocks = cdiv(most < a.few ? most : a.few, 8 * NT), items = blocks * a.kv_heads;
    OQ_REQUIRE(items <= 65535, "kv4_attention: too many key heads");
    const bool split = (int64_t)share > 16 * items * batch->sequences;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split ? 8 * NT : 1, (unsigned)items, batch->sequences);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t err = split ? cudaLaunchKernelEx(&cfg, join_kernel<T, HD, NT, true>, a, share)
                            : cudaLaunchKernelEx(&cfg, join_kernel<T, HD, NT, false>, a, share);
    if (err != cudaSuccess) {
        set_error("kv4_attention (join): launch failed: %s", cudaGetErrorString(err));
        return OQ_ERR_CUDA;
    }
    return OQ_OK;
}

template <typename T, int HD, int GS>
int stream_columns(Args &a, const oq_kv4_batch *batch, int nt, cudaStream_t st) {
    return nt == 1 ? stream_launch<T, HD, GS, 1>(a, batch, st) : stream_launch<T, HD, GS, 2>(a, batch, st);
}

template <typename T>
int attention_typed(Args &a, const oq_kv4_cache *c, const oq_kv4_batch *batch, int nt, cudaStream_t st) {
    if (c->head_dim == 64)
        return c->group_size == 32 ? stream_columns<T, 64, 32>(a, batch, nt, st)
                                   : stream_columns<T, 64, 64>(a, batch, nt, st);
    return c->group_size == 32   ? stream_columns<T, 128, 32>(a, batch, nt, st)
           : c->group_size == 64 ? stream_columns<T, 128, 64>(a, batch, nt, st)
                                 : stream_columns<T, 128, 128>(a, batch, nt, st);
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

extern "C" int64_t oq_kv4_attention_workspace_bytes(const oq_kv4_cache *cache, const oq_kv4_batch *batch,
                                                    int q_heads) {
    if (check_cache(cache) || check_batch(batch, 1) || check_heads(cache, q_heads)) return 0;
    const int nt = columns_of(cache, batch, q_heads);
    const int64_t share = nt == 1 ? share_of<1>() : share_of<2>();
    return (int64_t)header_bytes(batch) + share * 2 * 8 * nt * (cache->head_dim + 2) * 4;
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
    OQ_REQUIRE(scale == scale && scale - scale == 0.0f, "kv4_attention: scale must be finite");
    OQ_REQUIRE((int64_t)ws_bytes >= oq_kv4_attention_workspace_bytes(cache, batch, q_heads),
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
    a.q_heads = q_heads;
    a.ratio = q_heads / cache->kv_heads;
    a.f = scale * 1.4426950408889634f;
    a.window = window;
    a.causal = (flags & OQ_KV4_NOT_CAUSAL) ? 0 : 1;
    a.prefix = static_cast<int64_t *>(workspace);
    a.parts = reinterpret_cast<float *>(static_cast<char *>(workspace) + header_bytes(batch));
    a.vec = aligned(q, 16) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
    const int nt = columns_of(cache, batch, q_heads);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t most = (int64_t)batch->max_tokens * a.ratio;  // rows a sequence and key head
    a.few = a.ratio > kFew ? a.ratio : kFew;                   // single tokens are always streamed
    if (most > a.few) {
        // sum over sequences of ceil(rows / kPromptRows), at most
        const int64_t items = (cdiv(tokens * a.ratio, kPromptRows) + batch->sequences) * a.kv_heads;
        if (int rc = prompt_attention(a, dtype, cache, batch->sequences, items, st)) return rc;
    }
    return dtype == OQ_F16 ? attention_typed<__half>(a, cache, batch, nt, st)
                           : attention_typed<__nv_bfloat16>(a, cache, batch, nt, st);
}
