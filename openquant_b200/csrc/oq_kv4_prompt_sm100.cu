// Attention over the 4-bit key/value cache, many query rows per key head
// (chunks of prompts): both products on the tcgen05 tensor cores.
//
// Mathematics.  A CTA has 256 query rows of one key head -- rows are (token,
// query head of the key head) in that order, so all query heads that share a
// key head share its dequantization -- as two tiles of 128, and walks the
// cache in blocks of 128 tokens:
//     S = Q K^T (fp32 in TMEM),  p = 2^(S f - m),  O = O + P V
// with the running maximum m of a row raised only when a score passes it by
// 2^14 (see kRaise): then O, in TMEM, is multiplied by 2^(m_old - m_new);
// otherwise it is not touched.  K and V go to shared memory as code * scale,
// which are fp16 numbers exactly; P is rounded to fp16 (at most 2^14, largest
// at least 2^6) and goes back into S's TMEM columns as the second product's
// A operand.  Queries are fp16 (bf16 rows times a power of two).
//
// Roles: warps 0-3 and 4-7 are the softmax of the two tiles (a thread a row),
// warps 8-11 turn codes into fp16 tiles, warp 12 issues the products, warps
// 13-15 see beforehand whether all pages are there (the softmax then looks up
// no page: 165 us for 166 of ragged prompts with a word a block from the
// dequantizing warps).  While one tile's softmax runs, the other tile's
// products do: P0 V, Q0 K', P1 V, Q1 K', ...  The first half of a P is
// multiplied while the second is made.
//
// What bounds it.  For 4096 queries over 32768 tokens (64 query and 8 key
// heads, bf16): 3.11 ms, 1.32 PFLOP/s, 80 % of the measured dense bf16 rate,
// tensor pipe busy 64 % of the cycles.  A block of 256 rows costs about 3400
// cycles; the products alone take 2048 (64 cycles each, measured with
// everything else left out), the exponentials 2048 of the 16 a cycle that an
// SM makes, the operands and the dequantized tiles 2048 of shared memory: the
// three have to overlap through one S and one P per tile (512 TMEM columns:
// two S, two O).  Tried against that, and slower: blocks of 64 tokens with two
// S buffers a tile (the 64-column product reads Q too often, 48 cycles for 32:
// 5200 cycles for 128 tokens), eight dequantizing warps with S read twice for
// want of registers (4.1 ms), seven of them, three on V (3.4 ms), and CTAs that
// stay and fetch the next item's queries early, their items drawn from a
// counter (3.2 ms, but ragged prompts 198 us for 179 and a mixed step 352 us
// for 325).  What helped is noted where it is.
//
// At short contexts an item's own costs count: 1.7 us to find it and allocate
// TMEM, 3 us for the queries, 2.5 us for the output.
//
// Layouts: Q and K tiles are K-major, 128-byte swizzled, 64 elements a panel;
// V tiles have the same bytes (row = token) read as an MN-major operand.
// Within each eight elements of head_dim the order is that in which
// unpack_int() leaves a word's codes (0 4 1 5 2 6 3 7): the same for Q and K,
// and undone for V in the epilogue.
#include "oq_kv4_attention.cuh"

namespace oq {
namespace kv4 {
namespace {

constexpr int kThreads = 512;
constexpr int kTok = 128;        // cached tokens of a block
constexpr int kStages = 2;       // K tiles, and V tiles, in shared memory
constexpr int kLeastBlocks = 3;  // of a part of an item
constexpr uint32_t kTmemCols = 512;
// TMEM columns: the tiles' S (and P, in its first half) at 0 and 128, their O at 256 and 256 + head_dim
constexpr uint32_t kS = 0, kO = 256;
// Registers a thread: all warps start with kLaunchRegs; the dequantizing and
// the issuing warpgroup give some up (dec, never above what they have), the
// softmax warpgroups take them (inc, never below): a row of S is 128 of them.
// (With 184 and stores of 32 registers at a time the rows spilled: 5.1 ms
// where this takes 3.2.)
constexpr int kLaunchRegs = 65536 / kThreads, kSoftmaxRegs = 192, kDequantRegs = 88, kIssueRegs = 40;
static_assert(2 * kSoftmaxRegs + kDequantRegs + kIssueRegs <= 4 * kLaunchRegs, "register split");
static_assert(kSoftmaxRegs >= kLaunchRegs && kDequantRegs <= kLaunchRegs && kIssueRegs <= kLaunchRegs, "");

template <int HD>
struct Smem {
    static constexpr int kQPanel = 128 * 128, kPanel = kTok * 128;  // 64 elements of every row
    static constexpr int kQTile = kQPanel * (HD / 64), kTile = kPanel * (HD / 64);
    static constexpr int kQ = 0, kK = 2 * kQTile, kV = kK + kStages * kTile, kBars = kV + kStages * kTile;
    static constexpr int kBytes = kBars + 256 + 1024;  // barriers; slack to align to 1024
};

// tcgen05.mma B operand, MN-major, 128-byte swizzle: rows (k) of 64 elements,
// 8-row groups 1024 B apart, panels of 64 elements (mn) `panel` bytes apart.
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr, int panel) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(panel >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

template <int R>
__device__ __forceinline__ void regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

// One lane of a converged warp, in a form in which the compiler knows that the
// warp is converged: it then keeps the products' operands in uniform registers.
// (Issued behind `lane == 0` a product took 115 cycles instead of 89; a block
// of two tiles needs 2 (head_dim / 16 + 8) of them.)
__device__ __forceinline__ bool elect_one() {
    uint32_t v;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(v));
    return v != 0;
}

// 16 bytes that are read once: no line of the L1 is taken for them (beside
// 198 KB of shared memory it is small: with plain loads an item's queries took
// 10 us, so 3).
__device__ __forceinline__ uint4 ld16_once(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// mbar_wait() that looks at the clock and at the error word (a global load
// that all waiting warps of the GPU would share) only every 256th time; the
// hardware suspends a try for a while, so that stays far below the limit's
// resolution.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity) {
    const uint32_t a = smem_u32(bar);
    if (mbar_try_wait(a, parity)) return true;
    const long long t0 = clock64();
    for (int i = 1;; ++i) {
        if (mbar_try_wait(a, parity)) return true;
        if ((i & 255) == 0 && (clock64() - t0 > kWaitCycles || *(volatile int *)&g_device_error != 0)) {
            record_device_error(OQ_DEV_TIMEOUT);
            return false;
        }
    }
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The lowest n bits of a word; n may be below 0 or above 32.
__device__ __forceinline__ uint32_t ones(int n) { return n >= 32 ? 0xFFFFFFFFu : (1u << max(n, 0)) - 1; }

// Byte offset of the 16-byte chunk `c` (eight elements) of row r.
template <int PANEL>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return (uint32_t)((c >> 3) * PANEL + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void st16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// What item `id` (over all sequences with more than a.few rows that are not
// left out: the streaming work's joining kernel clears their rows) works on.
struct Item {
    int b, first, count, rows, head, row0;
    int length, base;   // cached tokens that can be read; position of the step's first token
    int nblk;       // blocks of kTok cached tokens from `lo` on, for all its parts
    int parts;      // parts it is cut into
    int floor, lo, hi;  // first visible token, the same down to 16, one past the last
};

// Finds it with all THREADS threads of the CTA; false: there is no such item.
template <int THREADS>
__device__ __forceinline__ bool find_item(const AttnArgs &a, int id, int cuts, Item &it) {
    __shared__ int warp_sum[THREADS / 32], found[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int base = 0;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    for (int b0 = 0; b0 < a.batch.sequences; b0 += THREADS) {
        const int b = b0 + tid;
        int n = 0;
        if (b < a.batch.sequences) {
            int first, count;
            const bool ok = tokens_of(a.batch, b, a.tokens, first, count);
            const int64_t rows = (int64_t)count * a.ratio;
            if (rows > a.few && ok && count <= a.max_tokens) n = (int)((rows + kPromptRows - 1) / kPromptRows) * a.kv_heads;
        }
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) warp_sum[warp] = inc;
        __syncthreads();
        int before = base;
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += warp_sum[w];
            base += warp_sum[w];
        }
        before += inc - n;
        if (id >= before && id < before + n) {
            found[0] = b;
            found[1] = id - before;
        }
        __syncthreads();
    }
    it.b = found[0];
    if (it.b < 0) return false;
    tokens_of(a.batch, it.b, a.tokens, it.first, it.count);
    int end;
    it.length = length_of(a.batch, it.b, a.page_size, end);
    it.base = end - it.count;
    it.rows = it.count * a.ratio;
    const int blocks = (it.rows + kPromptRows - 1) / kPromptRows;
    // the last rows see most: they go first
    it.head = found[1] % a.kv_heads;
    it.row0 = (blocks - 1 - found[1] / a.kv_heads) * kPromptRows;
    const int last = min(it.row0 + kPromptRows, it.rows) - 1;
    const int p0 = it.base + it.row0 / a.ratio, p1 = it.base + last / a.ratio;
    it.hi = a.causal ? min(p1 + 1, it.length) : it.length;
    it.floor = a.window > 0 ? (int)max((int64_t)p0 + 1 - a.window, (int64_t)0) : 0;
    it.lo = it.floor & ~15;
    it.nblk = it.hi > it.lo ? (it.hi - it.lo + kTok - 1) / kTok : 0;
    it.parts = max(min(cuts, it.nblk / kLeastBlocks), 1);
    return true;
}

// A part of an item: m[256], l[256], then O as float4 [HD / 4][256 rows]
// (columns in the order of TMEM).
template <int HD>
constexpr int kPartFloats = kPromptRows * (HD + 2);

template <typename T, int HD, int GS>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ AttnArgs a, int cuts) {
    using L = Smem<HD>;
    constexpr int NG = HD / GS, CH = HD / 32;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBars);
    // s_full: [tile]; p_full: [tile][half]; K and V: [stage]
    uint64_t *q_full = bars, *done = bars + 1, *s_full = bars + 2, *p_full = bars + 4, *k_full = bars + 8,
             *k_empty = k_full + kStages, *v_full = k_empty + kStages, *v_empty = v_full + kStages;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(v_empty + kStages);
    volatile uint32_t *holes_at = tmem_slot + 1;  // a token of this part has no page in the cache
    uint64_t *scanned = v_empty + kStages + 1;
    static_assert((8 + 4 * kStages) * 8 + 16 <= 256, "barrier space");
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

    asm volatile("griddepcontrol.launch_dependents;");  // the streaming kernel fills the SMs that run out of items
    Item it;
    const int part = blockIdx.x % cuts;
    if (!find_item<kThreads>(a, blockIdx.x / cuts, cuts, it) || part >= it.parts) return;
    const int b = it.b, first = it.first, length = it.length, rows = it.rows, head = it.head, row0 = it.row0;
    const int nrows = min(kPromptRows, rows - row0);
    const int base = it.base;
    // this part's blocks
    const int j0 = (int)((int64_t)part * it.nblk / it.parts), j1 = (int)((int64_t)(part + 1) * it.nblk / it.parts);
    const int nblk = j1 - j0;
    const int64_t floor = it.floor, lo = it.lo + (int64_t)j0 * kTok, hi = min(it.hi, it.lo + j1 * kTok);
    const int tiles = nrows > 128 ? 2 : 1;
    const int per = a.page_size >> 4;
    auto page_of = [&](int64_t t) {  // the page of token t; negative: none that is in the cache
        const int page = __ldg(a.batch.table + (int64_t)b * a.batch.max_pages + (int)(t >> 4) / per);
        return page < a.pages ? page : -1;
    };

    if (tid == 0) {
        mbar_init(q_full, 128 * tiles);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[2 * i], 128);
            mbar_init(&p_full[2 * i + 1], 128);
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&k_full[i], 128);
            mbar_init(&v_full[i], 128);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        mbar_init(done, 1);
        mbar_init(scanned, 96);
        *holes_at = 0;
        fence_barrier_init();
    }
    if (warp == 12) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp < 8) {
        // -------------------------------------------------------- softmax
        regs_inc<kSoftmaxRegs>();
        const int wg = warp >> 2, r = tid & 127;
        const int row = row0 + wg * 128 + r;
        const bool in = row < rows;
        if (wg < tiles) {
            const int tk = in ? row / a.ratio : 0;
            constexpr int LPR = HD / 8, PER = 32 / LPR;  // lanes a row, rows a step of the warp
            const int sub = lane / LPR, c = lane % LPR;
            // this thread's row in q (elements), and in the output and the log-sums (rows)
            const int64_t q_at = (int64_t)(first + tk) * a.q_ts +
                                 (int64_t)(head * a.ratio + (in ? row - tk * a.ratio : 0)) * a.q_hs;
            const int64_t at = (int64_t)(first + tk) * a.q_heads + head * a.ratio + (in ? row - tk * a.ratio : 0);
            const int live = min(max(rows - (row0 + wg * 128 + (warp & 3) * 32), 0), 32);  // rows of the warp
            float f = fabsf(a.f);
            {
                // The warp's 32 rows, PER at a time, a lane eight elements of one: whole
                // rows a load, all in flight.
                const uint32_t dst = smem_u32(smem + L::kQ + wg * L::kQTile);
                constexpr int U = 32 / PER;
                uint4 raw[U];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int n = i * PER + sub;
                    const int64_t from = __shfl_sync(0xffffffffu, (long long)q_at, n);
                    raw[i] = make_uint4(0, 0, 0, 0);
                    if (n < live) {
                        const T *src = static_cast<const T *>(a.q) + from + 8 * c;
                        if (a.vec) {
                            raw[i] = ld16_once(src);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) reinterpret_cast<T *>(&raw[i])[e] = src[e];
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float top = 0.0f, down, v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = Elem<T>::to_f32(reinterpret_cast<const T *>(&raw[i])[e]);
                    if (!std::is_same<T, __half>::value) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
#pragma unroll
                        for (int d = 1; d < LPR; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    }
                    float up = fp16_power<T>(top, down);
                    if (a.f < 0.0f) up = -up;
                    if (!std::is_same<T, __half>::value) {  // to the thread that has the row
                        down = __shfl_sync(0xffffffffu, down, lane % PER * LPR);
                        if (lane / PER == i) f *= down;
                    }
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = as_u32(__floats2half2_rn(v[e] * up, v[e + 4] * up));
                    st16(dst + chunk_at<L::kQPanel>((warp & 3) * 32 + i * PER + sub, c), w[0], w[1], w[2], w[3]);
                }
                fence_async_smem();
                mbar_arrive(q_full);
            }
            if (f == 0.0f) f = 1e-30f;  // masked scores are -inf before they are multiplied
            // tokens [low, vis) are what the row sees
            const int vis = a.causal ? min(base + tk + 1, length) : length;
            const int low = a.window > 0 ? (int)max((int64_t)base + tk + 1 - a.window, (int64_t)0) : 0;
            // tokens that every row of the tile sees
            const int last = min(row0 + wg * 128 + 127, rows - 1);
            const int all_vis = a.causal ? min(base + (row0 + wg * 128) / a.ratio + 1, length) : length;
            const int all_low = a.window > 0 ? (int)max((int64_t)base + last / a.ratio + 1 - a.window, (int64_t)0) : 0;
            const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t ts = tmem + quarter + kS + wg * kTok, to = tmem + quarter + kO + wg * HD;
            float m = kNone;
            float lim = -INFINITY, fe = f;  // m is raised above it; what s is multiplied with in p
            float2 l2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            bool ok = __all_sync(0xffffffffu, wait(scanned, 0));
            const bool holes = *holes_at != 0;
            for (int j = 0; ok && j < nblk; ++j) {
                ok = __all_sync(0xffffffffu, wait(&s_full[wg], j & 1));
                if (!ok) break;
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(ts + 32 * i, s[i]);
                tc_wait_ld();
                const int64_t t0 = lo + (int64_t)j * kTok;
                if (holes || t0 + kTok > all_vis || t0 < all_low) {
                    const int e0 = (int)min(max(low - t0, (int64_t)0), (int64_t)kTok);
                    const int e1 = (int)min(max(vis - t0, (int64_t)0), (int64_t)kTok);
                    uint32_t gone = 0;  // bit i: tokens 16 i .. of the block have no page
                    if (holes) {
#pragma unroll 1
                        for (int i = 0; i < kTok / 16; ++i)
                            if (t0 + 16 * i < hi && page_of(t0 + 16 * i) < 0) gone |= 1u << i;
                    }
                    // As words of 32 tokens, not by comparisons of each: ragged prompts 167 us
                    // with those (and two more loops' code for the pages), 156 with words.
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t seen = ones(e1 - 32 * w) & ~ones(e0 - 32 * w);
                        const uint32_t hide = ~seen | (gone >> 2 * w & 1) * 0xFFFFu | (gone >> (2 * w + 1) & 1) * 0xFFFF0000u;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (hide >> e & 1) s[w][e] = 0xff800000u;
                    }
                }
                float mx[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    mx[i] = __uint_as_float(s[i][0]);
#pragma unroll
                    for (int e = 1; e < 31; e += 2)
                        mx[i] = fmaxf(fmaxf(mx[i], __uint_as_float(s[i][e])), __uint_as_float(s[i][e + 1]));
                    mx[i] = fmaxf(mx[i], __uint_as_float(s[i][31]));
                }
                const float top = __fmul_rn(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), f);
                if (__any_sync(0xffffffffu, top > lim)) {
                    const float mn = top - m > kRaise ? top - kLift : m, corr = ex2(m - mn);
#pragma unroll
                    for (int i = 0; i < 2; ++i) l2[i].x *= corr, l2[i].y *= corr;
                    m = mn;
                    if (j > 0) {  // P V of the block before is complete: it was issued before this S
#pragma unroll 1
                        for (int i = 0; i < HD / 8; ++i) {
                            uint32_t o[8];
                            tmem_ld_32x32b_x8(to + 8 * i, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                            tmem_st_32x32b_x8(to + 8 * i, o);
                        }
                    }
                    // (a row that has passed kHuge, or has kNone, comes here with every block)
                    const bool huge = fabsf(m) > kHuge;
                    lim = huge ? -INFINITY : m + kRaise;
                    fe = huge ? 1.0f : f;
                    if (__any_sync(0xffffffffu, huge)) {
                        const float fm = huge ? f : 1.0f;
#pragma unroll
                        for (int i = 0; i < kTok; i += 2) {
                            const float2 x = __fmul2_rn(make_float2(__uint_as_float(s[i >> 5][i & 31]),
                                                                    __uint_as_float(s[i >> 5][(i & 31) + 1])),
                                                        make_float2(fm, fm));
                            s[i >> 5][i & 31] = __float_as_uint(x.x);
                            s[i >> 5][(i & 31) + 1] = __float_as_uint(x.y);
                        }
                    }
                }
                const float2 f2 = make_float2(fe, fe), m2 = make_float2(-m, -m);
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float2 x = __ffma2_rn(make_float2(__uint_as_float(s[h][2 * e]), __uint_as_float(s[h][2 * e + 1])),
                                              f2, m2);
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        l2[e & 1] = __fadd2_rn(l2[e & 1], x);
                        p[e] = as_u32(__floats2half2_rn(x.x, x.y));
                    }
                    tmem_st_32x32b_x16(ts + 16 * h, p);
                    if (h & 1) {  // half of P is ready: it is multiplied while the other half is made
                        tc_wait_st();
                        tc_fence_before();
                        mbar_arrive(&p_full[2 * wg + (h >> 1)]);
                    }
                }
            }
            const float l = (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
            // ------------------------------------------------- epilogue
            if (nblk > 0) {
                ok = __all_sync(0xffffffffu, ok && wait(done, 0));
                tc_fence_after();
            }
            if (ok && it.parts > 1) {
                float *dst = a.parts + (int64_t)blockIdx.x * kPartFloats<HD> + wg * 128 + r;
                dst[0] = m;
                dst[kPromptRows] = l;
                float4 *po = reinterpret_cast<float4 *>(a.parts + (int64_t)blockIdx.x * kPartFloats<HD> + 2 * kPromptRows) +
                             wg * 128 + r;
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(to + 32 * i, o);
                    tc_wait_ld();
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        po[(8 * i + x) * kPromptRows] =
                            make_float4(__uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]),
                                        __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3]));
                }
            } else if (ok) {
                // O / l through shared memory (Q's tile: every product is done), so that
                // whole rows go out
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const uint32_t mine = smem_u32(smem + L::kQ + wg * L::kQTile);
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    uint32_t o[32];
                    if (nblk > 0) {
                        tmem_ld_32x32b_x32(to + 32 * i, o);
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0;
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        alignas(16) T v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)  // column e holds element 0 4 1 5 2 6 3 7
                            put(&v[(e >> 1) + (e & 1) * 4], __uint_as_float(o[8 * x + e]) * inv);
                        const uint4 w = *reinterpret_cast<uint4 *>(v);
                        st16(mine + chunk_at<L::kQPanel>(r, 4 * i + x), w.x, w.y, w.z, w.w);
                    }
                }
                __syncwarp();
#pragma unroll 4
                for (int x = 0; x < 32; x += PER) {
                    const int rr = (warp & 3) * 32 + x + sub;
                    const int64_t to_row = __shfl_sync(0xffffffffu, (long long)at, x + sub);
                    uint4 w;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                                 : "r"(mine + chunk_at<L::kQPanel>(rr, c))
                                 : "memory");
                    if (x + sub < live)
                        *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + to_row * HD + 8 * c) = w;
                }
                if (in && a.log_sum != nullptr)
                    a.log_sum[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
            }
        }
        tc_fence_before();
        __syncthreads();
        return;  // each role ends by itself: the compiler then knows its register count
    }
    if (warp < 12) {
        // ---------------------------------------------------- dequantize
        regs_dec<kDequantRegs>();
        constexpr int N = kTok * CH / 128;  // 16-byte chunks of codes a thread takes of a K or V block
        constexpr int B16 = kTok / 16, kAhead = 32 / B16;  // 16-token rows of a block; blocks of one look-up
        const int r = tid & 127;
        // lane i: row / 16 in the cache of 16 tokens, from block `j` on, and which of
        // them have no page there.  Those stand at row 0 with scales of 0, and are masked.
        uint32_t row16 = 0, gone = 0;
        auto look_up = [&](int j) {
            row16 = 0;
            bool none = false;
            const int64_t t = lo + (int64_t)j * kTok + lane * 16;
            if (t < hi && t + 16 > floor) {
                const int page = page_of(t);
                none = page < 0;
                if (none)
                    index_error();
                else
                    row16 = (uint32_t)(((int64_t)page * a.kv_heads + head) * per + (int)(t >> 4) % per);
            }
            gone = __ballot_sync(0xffffffffu, none);
        };
        uint4 kc[N], vc[N];
        // Their scales, apart: whatever is done with a value in flight waits for it (packing
        // the two of a chunk into one register cost 1000 cycles a block).
        unsigned short ks[N], vs[N];
        // Chunk i of the thread: token r / CH + i * 128 / CH, 16-byte chunk r % CH, so
        // that all of them have one place within 16 tokens and one swizzle.
        const int tk0 = r / CH, c = r % CH;
        const size_t code_at = (size_t)(tk0 & 15) * (HD / 2) + c * 16, scale_at = (size_t)(tk0 & 15) * NG + c * 32 / GS;
        const uint8_t *k_lane = a.k_codes + code_at, *v_lane = a.v_codes + code_at;
        const unsigned short *ks_lane = reinterpret_cast<const unsigned short *>(a.k_scales) + scale_at;
        const unsigned short *vs_lane = reinterpret_cast<const unsigned short *>(a.v_scales) + scale_at;
        uint32_t r16[N];  // the chunks' rows / 16 in the cache, of the block that is loaded
        auto rows_of = [&](int j) {
            if (j >= nblk) return;
            if (j % kAhead == 0) look_up(j);
#pragma unroll
            for (int i = 0; i < N; ++i)
                r16[i] = __shfl_sync(0xffffffffu, row16, (j % kAhead) * B16 + ((tk0 + i * (128 / CH)) >> 4));
        };
        auto load = [&](int j, bool keys) {
            if (j >= nblk) return;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                // tokens that no row of the block sees may be anything: they become 0
                const int64_t t = lo + (int64_t)j * kTok + tk0 + i * (128 / CH);
                const bool live = t < hi && t >= floor;
                if (keys) {
                    kc[i] = ld16_once(k_lane + (size_t)r16[i] * (16 * HD / 2));
                    ks[i] = 0;
                    if (live) ks[i] = __ldg(ks_lane + (size_t)r16[i] * (16 * NG));
                } else {
                    vc[i] = ld16_once(v_lane + (size_t)r16[i] * (16 * HD / 2));
                    vs[i] = 0;
                    if (live) vs[i] = __ldg(vs_lane + (size_t)r16[i] * (16 * NG));
                }
            }
        };
        auto blank = [&](uint32_t gone_j, unsigned short (&sc)[N]) {  // bit i: tokens 16 i .. of the block
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (gone_j >> ((tk0 + i * (128 / CH)) >> 4) & 1) sc[i] = 0;
        };
        // the upper chunks of a row take their words in the order 2 3 0 1:
        // the eight lanes of a 128-byte store then hit different banks
        const bool swap = CH == 4 && (c & 2);
        const uint32_t tile_at = chunk_at<L::kPanel>(tk0, 4 * c + (swap ? 2 : 0));
        auto store = [&](uint32_t dst, const uint4 (&w)[N], const unsigned short (&sc)[N]) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const __half2 s2 = __half2half2(__ushort_as_half(sc[i]));
                const uint32_t word[4] = {swap ? w[i].z : w[i].x, swap ? w[i].w : w[i].y, swap ? w[i].x : w[i].z,
                                          swap ? w[i].y : w[i].w};
                const uint32_t at = dst + tile_at + i * (128 / CH * 128);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    __half2 v[4];
                    unpack_int(word[x], v);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __hmul2(v[e], s2);
                    // (x only flips bits of the chunk's place in its row, swizzled or not)
                    st16(at ^ (x << 4), as_u32(v[0]), as_u32(v[1]), as_u32(v[2]), as_u32(v[3]));
                }
            }
        };
        rows_of(0);
        load(0, true);
        load(0, false);
        bool ok = true;
        for (int j = 0; ok && j < nblk; ++j) {
            const int st = j % kStages, turn = j / kStages;
            if (turn > 0) ok = __all_sync(0xffffffffu, wait(&k_empty[st], (turn - 1) & 1));
            if (!ok) break;
            const uint32_t gone_j = gone >> (j % kAhead * B16);
            if (gone_j != 0) blank(gone_j, ks);
            store(smem_u32(smem + L::kK + st * L::kTile), kc, ks);
            fence_async_smem();
            mbar_arrive(&k_full[st]);
            rows_of(j + 1);
            load(j + 1, true);
            if (turn > 0) ok = __all_sync(0xffffffffu, wait(&v_empty[st], (turn - 1) & 1));
            if (!ok) break;
            if (gone_j != 0) blank(gone_j, vs);
            store(smem_u32(smem + L::kV + st * L::kTile), vc, vs);
            fence_async_smem();
            mbar_arrive(&v_full[st]);
            load(j + 1, false);
        }
        tc_fence_before();
        __syncthreads();
        return;
    }
    {
        // --------------------------------------------------------- issue
        regs_dec<kIssueRegs>();
        const int blocks_u = __shfl_sync(0xffffffffu, nblk, 0), tiles_u = __shfl_sync(0xffffffffu, tiles, 0);
        const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        if (warp == 12 && blocks_u > 0) {  // the whole warp walks, one lane issues
            constexpr uint32_t id_qk = umma_idesc_f16(128, kTok, false);
            constexpr uint32_t id_pv = umma_idesc_f16(128, HD, false) | 1u << 16;  // B is MN-major
            const uint32_t q0 = smem_u32(smem + L::kQ);
            auto scores = [&](int i, int j) {
                const uint64_t qd = umma_desc_sw128(q0 + i * L::kQTile);
                const uint64_t kd = umma_desc_sw128(smem_u32(smem + L::kK + (j % kStages) * L::kTile));
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k)
                        tc_mma_ss(tmem_u + kS + i * kTok, qd + ((uint64_t)((k >> 2) * L::kQPanel + (k & 3) * 32) >> 4),
                                  kd + ((uint64_t)((k >> 2) * L::kPanel + (k & 3) * 32) >> 4), id_qk, k != 0);
                    tc_commit(&s_full[i]);
                    if (i == tiles_u - 1) tc_commit(&k_empty[j % kStages]);
                }
                __syncwarp();
            };
            auto values = [&](int i, int j, int h) {
                const uint64_t vd = desc_mn_sw128(smem_u32(smem + L::kV + (j % kStages) * L::kTile), L::kPanel);
                if (elect_one()) {
#pragma unroll
                    for (int k = 4 * h; k < 4 * h + 4; ++k)
                        tc_mma_ts(tmem_u + kO + i * HD, tmem_u + kS + i * kTok + k * 8,
                                  vd + (uint64_t)(k * 16 * 128 >> 4), id_pv, j != 0 || k != 0);
                    if (h == 1 && i == tiles_u - 1) tc_commit(&v_empty[j % kStages]);
                }
                __syncwarp();
            };
            bool ok = wait(q_full, 0) && wait(&k_full[0], 0);
            if (ok) {
                tc_fence_after();
                for (int i = 0; i < tiles_u; ++i) scores(i, 0);
            }
            for (int j = 0; ok && j < blocks_u; ++j) {
                if (!(ok = wait(&v_full[j % kStages], (j / kStages) & 1))) break;
                for (int i = 0; i < tiles_u; ++i) {
                    if (!(ok = wait(&p_full[2 * i], j & 1))) break;
                    tc_fence_after();
                    values(i, j, 0);
                    if (!(ok = wait(&p_full[2 * i + 1], j & 1))) break;
                    tc_fence_after();
                    values(i, j, 1);
                    if (j + 1 < blocks_u) {
                        if (i == 0 && !(ok = wait(&k_full[(j + 1) % kStages], ((j + 1) / kStages) & 1))) break;
                        tc_fence_after();
                        scores(i, j + 1);
                    }
                }
            }
            // Every product this warp issued has completed once `done` fires.
            if (elect_one()) tc_commit(done);
            __syncwarp();
            wait(done, 0);
        }
        if (warp > 12) {  // are all pages there?  (while the queries are loaded)
            const int last = nblk > 0 ? (int)((hi - 1) >> 4) / per : -1;
            bool none = false;
#pragma unroll 4
            for (int p = (int)(max(lo, floor) >> 4) / per + (tid - 13 * 32); p <= last; p += 96)
                none |= page_of((int64_t)p * a.page_size) < 0;
            if (none) *holes_at = 1;
            mbar_arrive(scanned);
        }
        __syncwarp();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (warp == 12) tmem_dealloc(tmem, kTmemCols);
    }
}

// Adds the parts of the items that were cut: a thread a row, 16 columns a CTA.
template <typename T, int HD>
__global__ void __launch_bounds__(kPromptRows) join_prompt_kernel(const __grid_constant__ AttnArgs a, int cuts) {
    Item it;
    if (!find_item<kPromptRows>(a, blockIdx.x, cuts, it) || it.parts == 1) return;
    const int r = threadIdx.x, row = it.row0 + r;
    if (row >= it.rows) return;
    const float *src = a.parts + (int64_t)blockIdx.x * cuts * kPartFloats<HD> + r;
    float m = kNone, l = 0.0f;
    for (int p = 0; p < it.parts; ++p) m = fmaxf(m, src[(int64_t)p * kPartFloats<HD>]);
    float4 o[4] = {};
#pragma unroll 2
    for (int p = 0; p < it.parts; ++p) {
        const float *part = src + (int64_t)p * kPartFloats<HD>;
        const float c = ex2(part[0] - m);
        l = fmaf(c, part[kPromptRows], l);
        const float4 *po = reinterpret_cast<const float4 *>(part - r + 2 * kPromptRows) + blockIdx.y * 4 * kPromptRows + r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = po[i * kPromptRows];
            o[i].x = fmaf(c, v.x, o[i].x), o[i].y = fmaf(c, v.y, o[i].y);
            o[i].z = fmaf(c, v.z, o[i].z), o[i].w = fmaf(c, v.w, o[i].w);
        }
    }
    const int tk = row / a.ratio;
    const int64_t at = (int64_t)(it.first + tk) * a.q_heads + it.head * a.ratio + (row - tk * a.ratio);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *dst = static_cast<T *>(a.out) + at * HD + blockIdx.y * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // eight columns hold elements 0 4 1 5 2 6 3 7
        alignas(16) T v[8];
        const float4 x = o[2 * h], y = o[2 * h + 1];
        put(&v[0], x.x * inv), put(&v[4], x.y * inv), put(&v[1], x.z * inv), put(&v[5], x.w * inv);
        put(&v[2], y.x * inv), put(&v[6], y.y * inv), put(&v[3], y.z * inv), put(&v[7], y.w * inv);
        reinterpret_cast<uint4 *>(dst)[h] = *reinterpret_cast<uint4 *>(v);
    }
    if (blockIdx.y == 0 && a.log_sum != nullptr)
        a.log_sum[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <typename T, int HD, int GS>
int launch(const AttnArgs &a, int64_t items, int cuts, cudaStream_t st) {
    auto kern = prompt_kernel<T, HD, GS>;
    if (int rc = allow_dynamic_smem(reinterpret_cast<const void *>(kern), Smem<HD>::kBytes)) return rc;
    kern<<<(unsigned)(items * cuts), kThreads, Smem<HD>::kBytes, st>>>(a, cuts);
    if (int rc = check_launch("kv4_attention (prompt)")) return rc;
    if (cuts == 1) return OQ_OK;
    join_prompt_kernel<T, HD><<<dim3((unsigned)items, HD / 16), kPromptRows, 0, st>>>(a, cuts);
    return check_launch("kv4_attention (prompt join)");
}

template <typename T>
int launch_typed(const AttnArgs &a, const oq_kv4_cache *c, int64_t items, int cuts, cudaStream_t st) {
    if (c->head_dim == 64)
        return c->group_size == 32 ? launch<T, 64, 32>(a, items, cuts, st) : launch<T, 64, 64>(a, items, cuts, st);
    return c->group_size == 32   ? launch<T, 128, 32>(a, items, cuts, st)
           : c->group_size == 64 ? launch<T, 128, 64>(a, items, cuts, st)
                                 : launch<T, 128, 128>(a, items, cuts, st);
}

}  // namespace

// Into how many parts items are cut: what takes the GPU the fewest rounds of
// a part's blocks and its beginning and end (about kEnds blocks' time), for
// the longest context that the page table allows.
int prompt_cuts(const oq_kv4_cache *c, const oq_kv4_batch *b, int64_t items) {
    constexpr double kEnds = 5.0;
    const int64_t sms = sm_count(), blocks = cdiv((int64_t)b->max_pages * c->page_size, kTok);
    if (items >= 4 * sms) return 1;
    int best = 1;
    double least = 1e300;
    for (int n = 1; n <= kMostCuts && n <= blocks / kLeastBlocks + 1; ++n) {
        // a join costs about as much as a part's ends, too
        const double t = (double)cdiv(items * n, sms) * ((double)blocks / n + kEnds) + (n > 1 ? kEnds : 0.0);
        if (t < least) least = t, best = n;
    }
    return best;
}

int64_t prompt_part_bytes(const oq_kv4_cache *c, int64_t items, int cuts) {
    return cuts == 1 ? 0 : items * cuts * kPromptRows * (c->head_dim + 2) * 4;
}

int prompt_attention(const AttnArgs &a, int dtype, const oq_kv4_cache *c, int64_t items, int cuts, cudaStream_t st) {
    OQ_REQUIRE(items < (1ll << 31), "kv4_attention: too many query rows");
    return dtype == OQ_F16 ? launch_typed<__half>(a, c, items, cuts, st)
                           : launch_typed<__nv_bfloat16>(a, c, items, cuts, st);
}

}  // namespace kv4
}  // namespace oq
