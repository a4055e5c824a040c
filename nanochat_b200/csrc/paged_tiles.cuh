/*
 * k_paged_tiles: attention of at most 256 query slots (new rows of one request x the query heads of a key/value head), as two tiles of 128, over a run of the
 * request's pages, on tcgen05. A page's 64 keys at a time: S = Q K^T (M 128, N 64) into tensor memory, softmax in fp32 by four warps a tile, a row a
 * thread, the probabilities back over their scores, O += P V with P as the A operand from there; two S buffers a tile, so that the next page's scores run
 * under this page's softmax, and one tile's MMAs under the other's.
 *   - one block per SM with both tiles, which share the pages in its ring: what brings a page there (TMA, or widening it) is done once for 256 slots. Each tile
 *     has softmax warps and two that issue its MMAs, which go at their own pace; a page's place is free when both tiles have used it;
 *   - TWICE, where no request has more slots than one tile: both have the same, and every second page each. A page's chain of scores, softmax and products is long, and two
 *     of them run side by side (33 requests of 5 rows, 16 heads over 4, window 1,024: e4m3 42.3 -> 37.6 us, bf16 31.5 -> 28.8; behind whole contexts of up to 6,000
 *     positions 64.3 -> 66.5 and 43.9 -> 45.8; decided per piece instead, a prompt of 8,190 rows takes 254 us in place of 243, for the registers);
 *   - the block walks over the pieces of its part of the line (paged.cuh), the next piece's pages and queries coming under the end of this one;
 *   - the slots of a tile are packed by row and head, so that a chunk of few rows still fills the MMAs and a page is read
 *     once for all heads of its group; queries come as 3-d boxes (64 columns, the group's heads, a tile's rows);
 *   - pages are found through the block table; a page outside the pool is read as zeros and masked;
 *   - runs of pages, windows: rows may see nothing of a page at either end of their range, or nothing at all of a run;
 *   - probabilities are relative to a reference that need not be the maximum (the sum and O share it, so this is exact): a page's maximum is looked for only where a
 *     probability turns out above 2^7, or a row has seen nothing yet; then the reference is raised, O rescaled and the page done again;
 *   - bf16 pages: a probability enters P V as one bf16 term, at most 2^-9 of it away: the tensor cores would need 512 cycles a page and tile in place of
 *     256 for two terms;
 *   - e4m3 pages: four warps widen a quarter of every page each (a page each: drafts 55 us for 44) to f16 in shared memory (keys in the form of a TMA box, values transposed as they lie), in place
 *     of a launch that widens a request's pages into a workspace of twice the pool's size. Queries are made f16 once per piece, each row times a power of two.
 * Bound by the softmax warps' chain: a page of both tiles takes 2,000 cycles for bf16 pages, 1,300 of them on 64 exponentials a thread (the tensor cores need 1,000, and are 43 %
 * busy), the rest on tensor memory and barriers; 3,000 for e4m3, where 48 scale vectors a thread, the widened pages and the MMAs' operands share the shared memory's bandwidth.
 * 8,190 rows of a prompt, 16 heads over 4, bf16: 240 us, 1,145 TFLOP/s in short runs at 1,965 MHz (280 us where such calls fill seconds, and the card's power is bounded); 512 rows behind 16,384 positions,
 * 32 over 8: bf16 134 us (154), e4m3 193.
 * A position that a row does not see must not reach it: scores are masked, values are looked at in the pages that the border of some row crosses (three
 * at either end at most), and a page that holds one that is not finite there is multiplied row by row over the positions seen.
 */
#pragma once

#include "attn_tiles.cuh"
#include "paged.cuh"

namespace {
namespace tiles {

using namespace paged;
using att::arrive;

constexpr int ROWS = att::ROWS, KEYS = PAGE_TOKENS, TILE_WARPS = 4, SCORE_WARP = 2 * TILE_WARPS, VALUE_WARP = SCORE_WARP + 2, PAGE_WARP = VALUE_WARP + 2, PAGE_WARPS = 4;
constexpr int THREADS = 32 * (PAGE_WARP + PAGE_WARPS); /* four warps to a scheduler: 128 registers a thread */
constexpr float P_SCALE = 256.f, MIN_LOG2_VSCALE = -64.f;
constexpr int MOST_ODD = 8, HALF = KEYS / 2;
constexpr float C0 = 0.99992806f, C1 = 0.69326097f, C2 = 0.24261113f, C3 = 0.055171654f;
constexpr float LARGE = 128.f; /* how far a probability (bf16: the sum of a page's) may be above 1 before its row's reference is raised */
constexpr int TILE_COLUMNS = 256, AT_O = 2 * KEYS; /* tensor memory of a tile: S at 0 and 64, O at 128 */

template <bool E4M3> struct Shape {
    static constexpr int Q_BYTES = 2 * ROWS * 128, K_BYTES = 2 * KEYS * 128, V_BYTES = K_BYTES; /* Q: of a tile */
    static constexpr int STAGES = E4M3 ? 2 : 4, RAW_STAGES = E4M3 ? 4 : 0; /* raw: a page's bytes */
    static constexpr int AT_K = 2 * Q_BYTES, AT_V = AT_K + STAGES * K_BYTES, AT_RAW = AT_V + STAGES * V_BYTES, AT_SCALE = AT_RAW + RAW_STAGES * PAGE_BYTES;
    static constexpr int SCALE_FLOATS = 3 * KEYS, SCALES = 8, AT_BARS = AT_SCALE + (E4M3 ? SCALES * SCALE_FLOATS * 4 : 0);
    static constexpr int AT_HALF = AT_BARS + 1024, SMEM = 1024 + AT_HALF + ROWS * 8; /* half: the second tile's maxima and sums where both have the same slots */
    static_assert(SMEM <= 227 * 1024, "one block per SM");
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
/* 2^x of two values without the special-function unit: x' = sat((x + 125) / 250) keeps x in [-125, 125], x = n + f with n the nearest whole number (left in the
 * low bits of a sum with 1.5 * 2^23), 2^f by a cubic with least relative error on [-1/2, 1/2] (7.5e-5, a twentieth of what rounding to bf16 may
 * take), n added to its exponent. NaN counts as 0 (x = -125): who calls it looks for that. */
__device__ __forceinline__ void ex2_by_cubic(float &x, float &y, float score_x, float score_y, float slope, float offset) {
    float a, b;
    asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(a) : "f"(score_x), "f"(slope), "f"(offset));
    asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(b) : "f"(score_y), "f"(slope), "f"(offset));
    auto twice = [](float v) { return att::pair_of(v, v); };
    constexpr float MAGIC = 12582912.f - 125.f;
    float t0, t1, f0, f1;
    const uint64_t ab = att::pair_of(a, b);
    att::fma2(t0, t1, ab, twice(250.f), twice(MAGIC));
    att::fma2(f0, f1, att::pair_of(t0, t1), twice(-1.f), twice(MAGIC));
    att::fma2(f0, f1, ab, twice(250.f), att::pair_of(f0, f1));
    const uint64_t f = att::pair_of(f0, f1);
    att::fma2(x, y, f, twice(C3), twice(C2));
    att::fma2(x, y, att::pair_of(x, y), f, twice(C1));
    att::fma2(x, y, att::pair_of(x, y), f, twice(C0));
    x = __int_as_float(__float_as_int(x) + (__float_as_int(t0) << 23)), y = __int_as_float(__float_as_int(y) + (__float_as_int(t1) << 23));
}
__device__ __forceinline__ float log2_of(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t f16_pair(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

/* What the MMAs of a page do, by a warp: each thread its row's probabilities (from tensor memory, as the MMA would read them) times the values of
 * positions [from, seen), added to O. Rare. */
template <bool E4M3> __device__ __forceinline__ void multiply_seen(const uint8_t *v, uint32_t p_mine, uint32_t o_mine, int from, int seen, bool first) {
#pragma unroll 1
    for (int c = 0; c < HEAD_DIM / 16; c++) {
        float o[16] = {};
        if (!first) att::tmem_load16(o_mine + c * 16, o);
#pragma unroll 1
        for (int j = 0; j < KEYS / 2; j++) {
            const uint32_t x = att::tmem_word(p_mine + j);
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x));
            const float p[2] = {E4M3 ? f.x : __uint_as_float(x << 16), E4M3 ? f.y : __uint_as_float(x & 0xffff0000u)};
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (2 * j + k >= from && 2 * j + k < seen)
#pragma unroll
                    for (int e = 0; e < 16; e++) o[e] = fmaf(p[k], att::staged_value<E4M3>(v, 2 * j + k, c * 16 + e), o[e]);
        }
        __syncwarp();
        uint32_t x[16];
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = __float_as_uint(o[e]);
        att::tmem_store16(o_mine + c * 16, x);
    }
    att::tmem_wait_store();
}

/* A row of the query tile (two boxes of 64 columns, swizzled) from bf16 to f16 in place, times the power of two that brings its largest
 * magnitude to [2^14, 2^15); returns the factor that undoes it. */
__device__ __forceinline__ float query_row_to_f16(uint8_t *q, int row) {
    uint4 *chunk[2] = {reinterpret_cast<uint4 *>(q + row * 128), reinterpret_cast<uint4 *>(q + ROWS * 128 + row * 128)};
    float most = 0.f;
#pragma unroll 4
    for (int c = 0; c < 16; c++) { /* in the order that eight rows do not meet on a bank */
        const uint4 x = chunk[c >> 3][(c ^ row) & 7];
#pragma unroll
        for (int e = 0; e < 4; e++) most = fmaxf(most, fmaxf(fabsf(__uint_as_float((&x.x)[e] << 16)), fabsf(__uint_as_float((&x.x)[e] & 0xffff0000u))));
    }
    const int expo = (int)((__float_as_uint(most) >> 23) & 0xffu) - 127, down = max(-100, min(expo - 14, 112));
    const float mul = __uint_as_float((uint32_t)(127 - down) << 23);
#pragma unroll 4
    for (int c = 0; c < 16; c++) {
        uint4 *at = chunk[c >> 3] + ((c ^ row) & 7);
        uint4 x = *at;
#pragma unroll
        for (int e = 0; e < 4; e++) (&x.x)[e] = f16_pair(__uint_as_float((&x.x)[e] << 16) * mul, __uint_as_float((&x.x)[e] & 0xffff0000u) * mul);
        *at = x;
    }
    return __uint_as_float((uint32_t)(127 + down) << 23);
}

template <bool E4M3, bool TWICE> __global__ void __launch_bounds__(THREADS, 1) k_paged_tiles(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv,
                                                                                            const PagedArgs args) {
    using S = Shape<E4M3>;
    constexpr int STAGES = S::STAGES, RAW = E4M3 ? S::RAW_STAGES : 1;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t *raw = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const ncb_paged &a = args.p;
    const uint32_t base = smem_u32(raw), bars = base + S::AT_BARS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(raw + S::AT_BARS + 512);
    volatile int *failed = reinterpret_cast<volatile int *>(raw + S::AT_BARS + 520);
    volatile int *odd_of = reinterpret_cast<volatile int *>(raw + S::AT_BARS + 528); /* [2][MOST_ODD]: the b-th page that a tile's border crosses has b + 1 at b % MOST_ODD if a value is not finite */
    /* the k-th page of the block uses entry k % STAGES, the c-th page of a tile entry c % 2 */
    auto k_full = [&](int k) { return bars + 8u * (k % STAGES); };
    auto k_free = [&](int k) { return bars + 32u + 8u * (k % STAGES); };
    auto v_full = [&](int k) { return bars + 64u + 8u * (k % STAGES); };
    auto v_free = [&](int k) { return bars + 96u + 8u * (k % STAGES); };
    auto raw_full = [&](int k) { return bars + 128u + 8u * (k % RAW); };
    auto raw_free = [&](int k) { return bars + 320u + 8u * (k % RAW); };
    const uint32_t half_ready = bars + 352u; /* TWICE: the second tile's state */
    auto of_tile = [&](int x, int i) { return bars + 160u + 80u * x + 8u * i; };
    auto s_full = [&](int x, int c) { return of_tile(x, c & 1); };
    auto p_ready = [&](int x, int c) { return of_tile(x, 2 + (c & 1)); };
    auto pv_done = [&](int x, int c) { return of_tile(x, 4 + (c & 1)); };
    auto looked = [&](int x) { return of_tile(x, 6); };
    auto o_free = [&](int x) { return of_tile(x, 7); };
    auto q_full = [&](int x) { return of_tile(x, 8); };
    auto q_ready = [&](int x) { return of_tile(x, 9); }; /* E4M3: f16 */
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < 4; s++) {
            mbar_init(bars + 8u * s, E4M3 ? PAGE_WARPS : 1);
            mbar_init(bars + 32u + 8u * s, 2);
            mbar_init(bars + 64u + 8u * s, E4M3 ? PAGE_WARPS : 1);
            mbar_init(bars + 96u + 8u * s, 2);
            mbar_init(bars + 128u + 8u * s, 1);
            mbar_init(bars + 320u + 8u * s, PAGE_WARPS);
        }
        for (int x = 0; x < 2; x++) {
            for (int c = 0; c < 2; c++) {
                mbar_init(s_full(x, c), 1);
                mbar_init(p_ready(x, c), TILE_WARPS);
                mbar_init(pv_done(x, c), 1);
            }
            mbar_init(looked(x), TILE_WARPS);
            mbar_init(o_free(x), TILE_WARPS);
            mbar_init(q_full(x), 1);
            mbar_init(q_ready(x), TILE_WARPS);
        }
        mbar_init(half_ready, TILE_WARPS);
        *failed = 0;
        for (int i = 0; i < 2 * MOST_ODD; i++) odd_of[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    /* The block's pieces: where owners are whole, one of them, the longest first. */
    int piece, pieces;
    bool whole;
    {
        const Line line(args, 1);
        whole = line.whole;
        if (whole) {
            piece = line.n - 1 - (int)(blockIdx.x / line.heads), pieces = blockIdx.x < (long long)line.n * line.heads ? piece + 1 : piece;
        } else {
            const bool on = line.n > 0 && (int)blockIdx.x < args.caps.tile.blocks;
            piece = on ? line.starts[blockIdx.x].piece : 0, pieces = on ? line.starts[blockIdx.x + 1].piece : 0;
        }
    }
    if (piece >= pieces) return; /* nothing to do, before any tensor memory is taken */
    if (warp == SCORE_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    att::fence_before();
    __syncthreads();
    att::fence_after();
    const uint32_t tmem = *tmem_slot;
    const int rows_per = args.caps.tile.rows_per / 2; /* of a tile */
    auto wait = [&](uint32_t bar, int use) { /* one thread */
        if (att::mbar_test(bar, use & 1)) return true;
        if (!*failed && mbar_wait(bar, use & 1)) return true;
        flag(a.status, NCB_DEV_WAIT_TIMEOUT);
        *failed = 1;
        return false;
    };
    auto wait_all = [&](uint32_t bar, int use) { return (bool)__all_sync(0xffffffffu, wait(bar, use)); }; /* a warp */
    auto piece_at = [&](int piece) {
        const int *w = a.work + class_at(args.caps, 1);
        if (!whole) return reinterpret_cast<const Piece *>(w + pieces_at(args.caps.tile))[piece];
        const Owner o = reinterpret_cast<const Owner *>(w + HEADER_WORDS)[piece];
        return Piece{o.request, o.row, o.rows, o.pos, o.page0, o.pages, (int)blockIdx.x % a.Hkv, -1};
    };
    auto load_piece = [&] { return piece_at(piece); };
    auto begin_of = [&](int pos) { return a.window > 0 ? max(0, pos + 1 - a.window) : 0; };
    /* What tile x has of a piece: its rows and its first row's position; the pages that some row of it sees, from the piece's first; the border of some row's range
     * lies in the pages before lo and in those from hi on. TWICE: both tiles have the rows, and every second page each. `count` pages are the tile's. */
    constexpr int STEP = TWICE ? 2 : 1;
    struct Tile {
        int rows, pos, pages, count, lo, hi;
    };
    auto tile_of = [&](const Piece &e, int x) {
        Tile t;
        const int row0 = TWICE && e.pages > 0 ? 0 : x * rows_per;
        t.rows = max(0, min(rows_per, e.rows - row0)), t.pos = e.pos + row0;
        const int last = t.pos + t.rows - 1;
        t.pages = t.rows > 0 ? max(0, min(e.pages, last / KEYS + 1 - e.page0)) : 0;
        t.count = TWICE ? (t.pages + 1 - x) >> 1 : t.pages;
        t.lo = (begin_of(last) - e.page0 * KEYS + KEYS - 1) / KEYS, t.hi = (t.pos + 1) / KEYS - e.page0;
        return t;
    };
    auto takes = [&](const Tile &t, int x, int i) { return i < t.pages && (!TWICE || (i & 1) == x); };
    bool ok = true;

    if (warp >= PAGE_WARP) {
        if (!E4M3) {
            if (warp == PAGE_WARP && lane == 0) { /* copies keys and values */
                const uint64_t keep = policy_evict_last();
                int k = 0, v = 0; /* copies begun */
                for (; ok && piece < pieces; piece++) {
                    const Piece e = load_piece();
                    const int *table = a.table + (size_t)e.request * a.width + e.page0;
                    int page = e.pages > 0 ? table[0] : 0;
                    for (int i = 0; i < e.pages; i++) {
                        const int next = i + 1 < e.pages ? table[i + 1] : 0;
                        const bool in = (unsigned)page < (unsigned)a.n_pages;
                        if (!in) flag(a.status, NCB_DEV_BAD_PAGE);
                        /* outside the pool: a box behind its end, zeros */
                        const int row = in ? (page * a.Hkv + e.head) * 2 * KEYS : a.n_pages * a.Hkv * 2 * KEYS, st = k % STAGES;
                        /* The values of the page before in this place first: a softmax warp that has this page's scores may wait for its values' barrier next, by parity, and need not
                         * have waited for that page's (the other tile's, it may be, whose owner has no rows for this one) */
                        if (k >= STAGES && !(ok = wait(v_full(k), k / STAGES - 1))) break;
                        if (k >= STAGES && !(ok = wait(k_free(k), k / STAGES - 1))) break;
                        mbar_expect_tx(k_full(k), S::K_BYTES);
                        for (int j = 0; j < 2; j++) tma_load(base + S::AT_K + st * S::K_BYTES + j * KEYS * 128, &map_kv, 64 * j, row, k_full(k), keep);
                        k++;
                        if (v >= STAGES && !(ok = wait(v_free(v), v / STAGES - 1))) break;
                        mbar_expect_tx(v_full(v), S::V_BYTES);
                        for (int j = 0; j < 2; j++) tma_load(base + S::AT_V + st * S::V_BYTES + j * KEYS * 128, &map_kv, 64 * j, row + KEYS, v_full(v), keep);
                        v++;
                        page = next;
                    }
                }
                if (*failed) { /* the block must not leave under copies still in flight */
                    for (int i = max(0, k - STAGES); i < k; i++) mbar_wait(k_full(i), i / STAGES & 1);
                    for (int i = max(0, v - STAGES); i < v; i++) mbar_wait(v_full(i), i / STAGES & 1);
                }
            }
        } else { /* a quarter of every page is this warp's to widen: a place of the two is empty no longer than that takes. The first warp fetches pages */
            const int y = warp - PAGE_WARP;
            int fetch_piece = piece, fetch_at = 0, fetch_pages = -1, fetched = 0; /* the next page to fetch: its piece, its number there, and the block's pages before */
            long long fetch_table = 0;
            int fetch_head = 0;
            auto fetch = [&] {
                while (fetch_pages < 0 || fetch_at >= fetch_pages) {
                    if (fetch_pages >= 0) fetch_at = 0, fetch_piece++;
                    if (fetch_piece >= pieces) return;
                    const Piece e = piece_at(fetch_piece);
                    fetch_pages = e.pages, fetch_head = e.head, fetch_table = (long long)e.request * a.width + e.page0;
                }
                const int page = a.table[fetch_table + fetch_at];
                const bool in = (unsigned)page < (unsigned)a.n_pages;
                if (lane == 0) {
                    if (!in) flag(a.status, NCB_DEV_BAD_PAGE);
                    mbar_expect_tx(raw_full(fetched), PAGE_BYTES); /* outside the pool: page 0, masked and widened to zeros */
                    bulk_load(base + S::AT_RAW + fetched % RAW * PAGE_BYTES, (const uint8_t *)a.pool + ((size_t)(in ? page : 0) * a.Hkv + fetch_head) * PAGE_BYTES, PAGE_BYTES,
                              raw_full(fetched));
                }
                fetched++, fetch_at++;
            };
            if (y == 0)
                for (int i = 0; i < RAW; i++) fetch();
            int k = 0; /* the block's pages */
            for (; ok && piece < pieces; piece++) {
                const Piece e = load_piece();
                const int *table = a.table + (size_t)e.request * a.width + e.page0;
                int number = e.pages > 0 ? table[0] : 0;
                for (int i = 0; i < e.pages; i++, k++) {
                    const uint8_t *page = raw + S::AT_RAW + k % RAW * PAGE_BYTES;
                    const bool in = (unsigned)number < (unsigned)a.n_pages;
                    number = i + 1 < e.pages ? table[i + 1] : 0;
                    if (y == 0 && k > 0) { /* into the place of the page before, which all have read */
                        if (!(ok = wait_all(raw_free(k - 1), (k - 1) / RAW))) break;
                        fetch();
                    }
                    ok = wait_all(raw_full(k), k / RAW) && (k < STAGES || wait_all(k_free(k), k / STAGES - 1));
                    if (!ok) break;
                    uint8_t *keys = raw + S::AT_K + k % STAGES * S::K_BYTES;
                    uint4 in4[4];
                    float *scales = reinterpret_cast<float *>(raw + S::AT_SCALE) + k % S::SCALES * S::SCALE_FLOATS;
                    if (lane < 16) { /* score factor, log2 of the value's scale, its scale; with the keys, so that the softmax need not wait for the values' place. Page k - 8's have been read: the
                                    * scores of page k - 2 are there, and so the tile's buffers of two pages before that one were free */
                        const int j = 16 * y + lane;
                        const float vs = in ? reinterpret_cast<const float *>(page + PAGE_VS)[j] : 0.f;
                        scales[j] = in ? reinterpret_cast<const float *>(page + PAGE_KS)[j] : 0.f;
                        scales[KEYS + j] = fmaxf(log2_of(vs), MIN_LOG2_VSCALE);
                        scales[2 * KEYS + j] = vs * P_SCALE;
                    }
#pragma unroll
                    for (int n = 0; n < 4; n++) in4[n] = *reinterpret_cast<const uint4 *>(page + page_k_chunk(16 * y + 4 * n + (lane >> 3), lane & 7)); /* 16 codes of a key */
#pragma unroll
                    for (int n = 0; n < 4; n++) { /* -> 32 bytes: two chunks of a swizzled row */
                        const int j = 16 * y + 4 * n + (lane >> 3), c = lane & 7;
                        uint4 w[2];
                        widen_e4m3x4(in4[n].x, w[0].x, w[0].y), widen_e4m3x4(in4[n].y, w[0].z, w[0].w);
                        widen_e4m3x4(in4[n].z, w[1].x, w[1].y), widen_e4m3x4(in4[n].w, w[1].z, w[1].w);
                        uint8_t *row = keys + (c >> 2) * KEYS * 128 + j * 128;
                        const uint32_t chunk = ((2 * c & 7) ^ (j & 7)) << 4;
                        *reinterpret_cast<uint4 *>(row + chunk) = w[0];
                        *reinterpret_cast<uint4 *>(row + (chunk ^ 16)) = w[1];
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) arrive(k_full(k));
#pragma unroll
                    for (int n = 0; n < 4; n++) in4[n] = *reinterpret_cast<const uint4 *>(page + PAGE_V + y * 2048 + (n * 32 + lane) * 16); /* 16 positions of a dimension */
                    if (k >= STAGES && !(ok = wait_all(v_free(k), k / STAGES - 1))) break;
                    uint8_t *values = raw + S::AT_V + k % STAGES * S::V_BYTES;
                    const int used = (in ? e.pos + e.rows - (e.page0 + i) * KEYS : 0) - 16 * y; /* positions past the last row may hold anything: zeros */
                    if (used < 16) {
#pragma unroll
                        for (int n = 0; n < 4; n++)
#pragma unroll
                            for (int w = 0; w < 4; w++) {
                                const int on = used - 4 * w;
                                (&in4[n].x)[w] = on >= 4 ? (&in4[n].x)[w] : on <= 0 ? 0u : (&in4[n].x)[w] & ((1u << (8 * on)) - 1u);
                            }
                    }
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        uint4 w[2];
                        widen_e4m3x4(in4[n].x, w[0].x, w[0].y), widen_e4m3x4(in4[n].y, w[0].z, w[0].w);
                        widen_e4m3x4(in4[n].z, w[1].x, w[1].y), widen_e4m3x4(in4[n].w, w[1].z, w[1].w);
                        uint8_t *row = values + (n * 32 + lane) * 128;
                        const uint32_t chunk = (2 * y ^ (lane & 7)) << 4;
                        *reinterpret_cast<uint4 *>(row + chunk) = w[0];
                        *reinterpret_cast<uint4 *>(row + (chunk ^ 16)) = w[1];
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) arrive(v_full(k)), arrive(raw_free(k));
                }
            }
            if (*failed && y == 0 && lane == 0) /* the block must not leave under copies still in flight */
                for (int i = max(0, fetched - RAW); i < fetched; i++) mbar_wait(raw_full(i), i / RAW & 1);
        }
    } else if (warp >= SCORE_WARP) { /* a tile's MMAs, scores and values each by a warp of their own (issuing them and the waits between take longer than the tensor
                                        * cores need); it goes through the loop together (elect_one) */
        constexpr uint32_t F32 = 1u << 4, BF16_AB = E4M3 ? 0u : (1u << 7) | (1u << 10), M = (uint32_t)(ROWS >> 4) << 24;
        constexpr uint32_t score = F32 | BF16_AB | M | ((uint32_t)(KEYS >> 3) << 17);
        constexpr uint32_t value = F32 | BF16_AB | M | ((uint32_t)(HEAD_DIM >> 3) << 17) | (E4M3 ? 0u : 1u << 16);
        const int x = __shfl_sync(0xffffffffu, (warp - SCORE_WARP) & 1, 0);
        const uint32_t t = __shfl_sync(0xffffffffu, tmem, 0) + x * TILE_COLUMNS, b = __shfl_sync(0xffffffffu, base, 0);
        int k = 0, c = 0, used = 0, borders = 0; /* pages, pages of the tile, pieces that the tile had pages of, pages that its border crossed */
        int asked = 0, issued = 0;               /* copies of queries, pages whose MMAs this warp has begun */
        for (; ok && piece < pieces; piece++) {
            const Piece e = load_piece();
            if (e.pages == 0) continue;
            const Tile tile = tile_of(e, x);
            if (warp < VALUE_WARP) {
                if (tile.count > 0) { /* its queries, when the products of the piece before have read theirs */
                    if (used > 0 && !(ok = wait_all(s_full(x, c - 1), (c - 1) >> 1))) break;
                    if (elect_one()) {
                        const int group = a.Hq / a.Hkv;
                        mbar_expect_tx(q_full(x), 2 * rows_per * group * 128); /* a box is whole, whatever the tile uses of it */
                        for (int j = 0; j < 2; j++) tma_load_3d(b + x * S::Q_BYTES + j * ROWS * 128, &map_q, 64 * j, e.head * group, e.row + (TWICE ? 0 : x * rows_per), q_full(x));
                    }
                    asked = used + 1;
                    __syncwarp();
                    if (!(ok = wait_all(E4M3 ? q_ready(x) : q_full(x), used))) break;
                }
                for (int i = 0; ok && i < e.pages; i++, k++) {
                    ok = wait_all(k_full(k), k / STAGES);
                    if (!ok) break;
                    if (!takes(tile, x, i)) { /* the tile has no part in the page, which only passes */
                        if (lane == 0) arrive(k_free(k));
                        continue;
                    }
                    const int ci = c + i / STEP;
                    ok = ci < 2 || wait_all(pv_done(x, ci), (ci - 2) >> 1); /* the buffer's probabilities have been used */
                    if (!ok) break;
                    att::fence_after();
                    const uint32_t ks = b + S::AT_K + k % STAGES * S::K_BYTES, qs = b + x * S::Q_BYTES, d = t + (ci & 1) * KEYS;
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int h = 0; h < 4; h++)
                                umma_bf16(d, umma_desc(qs + j * ROWS * 128 + h * 32), umma_desc(ks + j * KEYS * 128 + h * 32), score, (j | h) != 0);
                        umma_commit(s_full(x, ci));
                        umma_commit(k_free(k));
                    }
                    issued = ci + 1;
                    __syncwarp();
                }
            } else {
                for (int i = 0; ok && i < e.pages; i++, k++) {
                    ok = wait_all(v_full(k), k / STAGES);
                    if (!ok) break;
                    if (!takes(tile, x, i)) {
                        if (lane == 0) arrive(v_free(k));
                        continue;
                    }
                    const int ci = c + i / STEP;
                    ok = (i >= STEP || used == 0 || wait_all(o_free(x), used - 1)) && wait_all(p_ready(x, ci), ci >> 1);
                    if (!ok) break;
                    att::fence_after();
                    const uint32_t vs = b + S::AT_V + k % STAGES * S::V_BYTES, p = t + (ci & 1) * KEYS;
                    bool by_mma = true;
                    if (i < tile.lo || i >= tile.hi) by_mma = odd_of[x * MOST_ODD + borders % MOST_ODD] != borders + 1, borders++;
                    if (elect_one()) {
                        if (by_mma) {
#pragma unroll
                            for (int h = 0; h < KEYS / 16; h++) /* 16 keys: 8 columns of packed probabilities */
                                att::umma_from_tmem(t + AT_O, p + h * 8, E4M3 ? umma_desc(vs + h * 32) : att::desc_by_rows(vs + h * 2048, KEYS * 128), value, (i / STEP | h) != 0);
                        }
                        umma_commit(pv_done(x, ci));
                        umma_commit(v_free(k));
                    }
                    issued = ci + 1;
                    __syncwarp();
                }
            }
            c += tile.count, used += tile.count > 0;
        }
        /* the block must not leave under a copy or MMAs still in flight: after a failed wait they may be, else they have long ended */
        if (asked > 0) mbar_wait(q_full(x), (asked - 1) & 1);
        if (issued > 0) mbar_wait(warp < VALUE_WARP ? s_full(x, issued - 1) : pv_done(x, issued - 1), ((issued - 1) >> 1) & 1);
    } else { /* softmax: a thread has a slot of its tile */
        const int x = warp / TILE_WARPS, slot = tid % (32 * TILE_WARPS), first = slot & ~31;
        const uint32_t t_mine = tmem + x * TILE_COLUMNS + ((uint32_t)first << 16), o_mine = t_mine + AT_O;
        int k = 0, c = 0, used = 0, borders = 0, joined = 0; /* joined: pieces of which both tiles had pages */
        for (; ok && piece < pieces; piece++) {
            const Piece e = load_piece();
            const Tile tile = tile_of(e, x);
            const int G = a.Hq / a.Hkv, slots = tile.rows * G, mine = min(slot, slots - 1) / G; /* the thread's row of the tile */
            const bool on = slot < slots;
            bf16 *out = (bf16 *)a.out + (size_t)(e.row + (TWICE && e.pages > 0 ? 0 : x * rows_per) + (on ? mine : 0)) * a.ldo + (size_t)(e.head * G + (on ? slot % G : 0)) * HEAD_DIM;
            if (e.pages == 0) { /* rows that are not served */
                if (on)
                    for (int d = 0; d < HEAD_DIM; d += 8) *reinterpret_cast<uint4 *>(out + d) = make_uint4(0u, 0u, 0u, 0u);
                continue;
            }
            float *part = (float *)a.workspace + parts_at(args.caps, 1) + ((size_t)max(e.part, 0) * args.caps.tile.slots + (TWICE ? 0 : x * rows_per * G) + slot) * PART;
            if (tile.count == 0) { /* the tile has no part in this piece: an empty state */
                if (!TWICE && on && e.part >= 0) part[0] = -INFINITY, part[1] = 0.f;
                k += e.pages;
                continue;
            }
            float factor = args.scale_log2;
            if (E4M3) { /* the thread's row to f16 */
                if (!(ok = wait_all(q_full(x), used))) break;
                factor *= query_row_to_f16(raw + x * S::Q_BYTES, slot);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(q_ready(x));
            }
            used++;
            const int last = tile.pos + mine - e.page0 * KEYS, begin = begin_of(tile.pos + mine) - e.page0 * KEYS; /* what the slot sees, from the piece's first key */
            /* the border of some row of the warp lies in the pages before my_lo and in those from my_hi on */
            const int my_lo = (__shfl_sync(0xffffffffu, begin, 31) + KEYS - 1) / KEYS, my_hi = (__shfl_sync(0xffffffffu, last, 0) + 1) / KEYS;
            const bool idle = first >= slots; /* a warp without a slot only keeps the others company */
            const int *table = a.table + (size_t)e.request * a.width + e.page0;
            const uint64_t factor2 = att::pair_of(factor, factor);
            float m = -INFINITY;
            uint64_t sums[2] = {0, 0};
            int page = table[TWICE ? x : 0];
            for (int i = TWICE ? x : 0; i < tile.pages; i += STEP) {
                const bool in = (unsigned)page < (unsigned)a.n_pages;
                page = i + STEP < tile.pages ? table[i + STEP] : 0;
                const int ci = c + i / STEP, ki = k + i;
                ok = wait_all(s_full(x, ci), ci >> 1);
                if (!ok) break;
                att::fence_after();
                const uint32_t s_mine = t_mine + (ci & 1) * KEYS;
                const float *scales = reinterpret_cast<const float *>(raw + S::AT_SCALE) + ki % S::SCALES * S::SCALE_FLOATS;
                auto scales_at = [&](int j, int which) { return *reinterpret_cast<const ulonglong2 *>(scales + which * KEYS + j); }; /* of four keys from j */
                const bool border = i < tile.lo || i >= tile.hi;
                const bool plain = i >= my_lo && i < my_hi && in; /* every row of the warp sees the whole page */
                if (!idle) {
                    uint32_t packed[KEYS / 2]; /* probabilities */
                    uint64_t sum[2];
                    constexpr bool CUBIC = !E4M3;
                    auto load_scores = [&](int h, float *s) { /* of half the page's keys, those from h on */
                        tmem_load32(s_mine + h, s);
                        if (E4M3) {
#pragma unroll
                            for (int j = 0; j < HALF; j += 4) {
                                const ulonglong2 f = scales_at(h + j, 0);
                                att::mul2(s[j], s[j + 1], att::pair_of(s[j], s[j + 1]), f.x);
                                att::mul2(s[j + 2], s[j + 3], att::pair_of(s[j + 2], s[j + 3]), f.y);
                            }
                        }
                        if (!plain) {
                            const int to = in ? last - i * KEYS - h : -1, from = begin - i * KEYS - h;
#pragma unroll
                            for (int j = 0; j < HALF; j++) s[j] = j > to || j < from ? -INFINITY : s[j];
                        }
                    };
                    auto probabilities = [&](bool cubic) { /* whether some is large */
                        const float reference = m == -INFINITY ? 0.f : m; /* where nothing counts yet the scores are -infinity or NaN: nothing, or NaN */
                        const uint64_t minus = att::pair_of(-reference, -reference);
                        const float slope = factor * (1.f / 250.f), offset = (125.f - reference) * (1.f / 250.f);
                        __half2 most = __floats2half2_rn(0.f, 0.f);
                        sum[0] = sum[1] = 0;
#pragma unroll
                        for (int h = 0; h < KEYS; h += HALF) {
                            float s[HALF];
                            load_scores(h, s);
#pragma unroll
                            for (int j = 0; j < HALF; j += 4) {
                                ulonglong2 f;
                                if (E4M3) f = scales_at(h + j, 2);
#pragma unroll
                                for (int p = 0; p < 2; p++) {
                                    float y, z;
                                    if (cubic && j % 8 == 4 && p == 1) { /* scores 6 and 7 of eight: the special-function unit would need 1,024 cycles a page for both tiles with all */
                                        ex2_by_cubic(y, z, s[j + 2], s[j + 3], slope, offset);
                                    } else {
                                        att::fma2(y, z, att::pair_of(s[j + 2 * p], s[j + 2 * p + 1]), factor2, minus);
                                        y = ex2(y), z = ex2(z);
                                    }
                                    const uint64_t yz = att::pair_of(y, z);
                                    sum[p] = att::add2(sum[p], yz);
                                    if (E4M3) {
                                        att::mul2(y, z, yz, p ? f.y : f.x);
                                        const __half2 w = __floats2half2_rn(y, z);
                                        most = __hmax2_nan(most, w);
                                        packed[(h + j) / 2 + p] = *reinterpret_cast<const uint32_t *>(&w);
                                    } else {
                                        const __nv_bfloat162 w = __floats2bfloat162_rn(y, z);
                                        packed[(h + j) / 2 + p] = *reinterpret_cast<const uint32_t *>(&w);
                                    }
                                }
                            }
                            if (cubic) { /* to saturate makes NaN zero: where one of these scores is not finite the sum becomes NaN, and the page is done again without the cubic
                                          * (here, off the loop's chains: prompts of 8,190 rows back to back 253.6 -> 254.6 us; beside each pair 259.2) */
                                const uint64_t some = att::add2(att::add2(att::pair_of(s[6], s[7]), att::pair_of(s[14], s[15])), att::add2(att::pair_of(s[22], s[23]), att::pair_of(s[30], s[31])));
                                sum[0] = att::add2(sum[0], att::mul2(some, 0));
                            }
                        }
                        if (E4M3) return !(__low2float(most) <= LARGE * P_SCALE && __high2float(most) <= LARGE * P_SCALE);
                        const uint64_t both = att::add2(sum[0], sum[1]);
                        return !(__uint_as_float((uint32_t)both) + __uint_as_float((uint32_t)(both >> 32)) <= LARGE);
                    };
                    /* Probabilities against the reference that holds, without looking for the page's maximum: only where one (or their sum) turns out above 2^7, or nothing
                     * holds yet, is it looked for and the page done again, for the rows that need it. */
                    const bool raise = on & ((CUBIC && plain ? probabilities(true) : probabilities(false)) | (m == -INFINITY));
                    if (__any_sync(0xffffffffu, raise)) {
                        float best[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
                        for (int h = 0; h < KEYS; h += HALF) {
                            float s[HALF];
                            load_scores(h, s);
#pragma unroll
                            for (int j = 0; j < HALF; j += 4) {
                                float y[4] = {s[j], s[j + 1], s[j + 2], s[j + 3]};
                                if (E4M3) { /* the probabilities carry the value's scale: the maximum is that of score + log2(scale) */
                                    const ulonglong2 f = scales_at(h + j, 1);
                                    att::fma2(y[0], y[1], att::pair_of(y[0], y[1]), factor2, f.x);
                                    att::fma2(y[2], y[3], att::pair_of(y[2], y[3]), factor2, f.y);
                                }
                                best[0] = att::max3(best[0], y[0], y[1]);
                                best[1] = att::max3(best[1], y[2], y[3]);
                            }
                        }
                        float top = fmaxf(best[0], best[1]);
                        if (!E4M3) top *= factor;
                        const bool grown = raise && top > m;
                        if (i >= STEP && __any_sync(0xffffffffu, grown)) {
                            ok = wait_all(pv_done(x, ci - 1), (ci - 1) >> 1); /* O is complete up to the page before */
                            if (!ok) break;
                            att::fence_after();
                            const float f = !grown ? 1.f : m == -INFINITY ? 0.f : ex2(m - top);
                            sums[0] = att::mul2(sums[0], att::pair_of(f, f)), sums[1] = att::mul2(sums[1], att::pair_of(f, f));
#pragma unroll 1
                            for (int d = 0; d < HEAD_DIM; d += 16) {
                                float y[16];
                                uint32_t z[16];
                                att::tmem_load16(o_mine + d, y);
#pragma unroll
                                for (int j = 0; j < 16; j++) z[j] = __float_as_uint(y[j] * f);
                                att::tmem_store16(o_mine + d, z);
                            }
                        }
                        m = grown ? top : m;
                        probabilities(false);
                    }
                    sums[0] = att::add2(sums[0], sum[0]), sums[1] = att::add2(sums[1], sum[1]);
                    att::tmem_store16(s_mine, packed);
                    att::tmem_store16(s_mine + KEYS / 4, packed + KEYS / 4);
                }
                if (border) {
                    ok = wait_all(v_full(ki), ki / STAGES);
                    if (!ok) break;
                    uint8_t *v = raw + S::AT_V + ki % STAGES * S::V_BYTES;
                    const int used = E4M3 ? KEYS : e.pos + e.rows - (e.page0 + i) * KEYS; /* positions past the last row may hold anything: zeros (E4M3: they are) */
                    bool strange = E4M3 && slot < KEYS && !isfinite(scales[2 * KEYS + slot]);
#pragma unroll 2
                    for (int y = slot; y < 2 * KEYS * 8; y += 32 * TILE_WARPS) {
                        uint4 *chunk = reinterpret_cast<uint4 *>(v) + y;
                        if (E4M3 || y / 8 % KEYS < used) strange |= att::not_finite8<E4M3>(*chunk);
                        else *chunk = make_uint4(0u, 0u, 0u, 0u);
                    }
                    if (!E4M3) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    strange = __any_sync(0xffffffffu, strange);
                    if (lane == 0) {
                        if (strange) odd_of[x * MOST_ODD + borders % MOST_ODD] = borders + 1;
                        arrive(looked(x));
                    }
                }
                if (!idle) att::tmem_wait_store();
                att::fence_before();
                __syncwarp();
                if (border) {
                    ok = wait_all(looked(x), borders);
                    if (!ok) break;
                    if (odd_of[x * MOST_ODD + borders % MOST_ODD] == borders + 1) {
                        /* O is complete up to the page before, or has been read (TWICE: by the other tile's warps, it may be) */
                        ok = i >= STEP ? wait_all(pv_done(x, ci - 1), (ci - 1) >> 1) : !TWICE || used < 2 || wait_all(o_free(x), used - 2);
                        if (!ok) break;
                        att::fence_after();
                        multiply_seen<E4M3>(raw + S::AT_V + ki % STAGES * S::V_BYTES, s_mine, o_mine, begin - i * KEYS, last - i * KEYS + 1, i < STEP);
                        att::fence_before();
                        __syncwarp();
                    }
                    borders++;
                }
                if (lane == 0) arrive(p_ready(x, ci));
            }
            ok = ok && wait_all(pv_done(x, c + tile.count - 1), (c + tile.count - 1) >> 1);
            if (!ok) break;
            att::fence_after();
            const uint64_t two = att::add2(sums[0], sums[1]);
            float l = __uint_as_float((uint32_t)two) + __uint_as_float((uint32_t)(two >> 32)), f = 1.f, f_other = 0.f;
            const bool join = TWICE && tile.pages > 1;
            if (join) { /* the first tile takes the second one's state, whose O it reads in tensor memory */
                float2 *half = reinterpret_cast<float2 *>(raw + S::AT_HALF);
                if (x == 1) {
                    half[slot] = make_float2(m, l);
                    att::fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(half_ready);
                    k += e.pages, c += tile.count, joined++;
                    continue;
                }
                ok = wait_all(half_ready, joined++);
                if (!ok) break;
                att::fence_after();
                const float2 other = half[slot];
                auto scale_of = [](float m, float l, float top) { return m == -INFINITY && l == l ? 0.f : ex2(m - top); }; /* nothing where the state holds nothing */
                const float top = fmaxf(m, other.x);
                f = scale_of(m, l, top), f_other = scale_of(other.x, other.y, top);
                l = l * f + other.y * f_other, m = top;
            }
            const float inv = l > 0.f || l != l ? __fdiv_rn(1.f, E4M3 ? l * P_SCALE : l) : 0.f;
            if (on && e.part >= 0) part[0] = m, part[1] = l;
#pragma unroll 1
            for (int d = 0; d < HEAD_DIM; d += 32) {
                float y[32];
                tmem_load32(o_mine + d, y);
                if (join) {
#pragma unroll
                    for (int h = 0; h < 32; h += 16) {
                        float z[16];
                        att::tmem_load16(o_mine + TILE_COLUMNS + d + h, z);
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const float own = f != 0.f ? y[h + j] * f : 0.f;
                            y[h + j] = f_other != 0.f ? fmaf(z[j], f_other, own) : own;
                        }
                    }
                }
                if (!on) continue;
                if (e.part < 0) {
                    att::store32(out + d, y, [&](int) { return inv; });
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(part + 4 + d + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
                }
            }
            att::fence_before();
            __syncwarp();
            if (lane == 0) {
                arrive(o_free(x));
                if (join) arrive(o_free(1));
            }
            k += e.pages, c += tile.count;
        }
    }
    att::fence_before();
    __syncthreads();
    if (warp == SCORE_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

} /* namespace tiles */
} /* namespace */
