/*
 * k_paged_tiles: attention of a tile of at most 128 query slots (new rows of one request x the query heads of a key/value head) over a run of
 * the request's pages, on tcgen05. A page's 64 keys at a time, as attn_tiles.cuh has it: S = Q K^T (M 128, N 64) into tensor memory, softmax in fp32 by
 * eight warps, the probabilities back over their scores, O += P V from there; two S buffers, so that the next page's scores run under
 * this page's softmax, and two blocks per SM. What is different here:
 *   - a block walks over the pieces of its part of the line (paged.cuh); the next piece's pages and queries come under the end of this one;
 *   - the slots of a tile are packed by row and head, so that a chunk of few rows still fills the MMAs and a page is read
 *     once for all heads of its group; queries come as 3-d boxes (64 columns, the group's heads, the tile's rows);
 *   - pages are found through the block table; a page outside the pool is read as zeros and masked;
 *   - runs of pages, windows: rows may see nothing of a page at either end of their range, or nothing at all of a run;
 *   - bf16 pages: a probability enters P V as one bf16 term, at most 2^-9 of it away: the tensor cores would need 512 cycles a page in place of
 *     256 for two terms;
 *   - e4m3 pages: two warps widen a page to f16 in shared memory (keys in the form of a TMA box, values transposed as they lie), in place of a launch that
 *     widens a request's pages into a workspace of twice the pool's size. Queries are made f16 once per piece, each row times a power of two.
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

constexpr int ROWS = att::ROWS, KEYS = PAGE_TOKENS, TILE_WARPS = 8, COPY_WARP = 8, MMA_WARP = 9, WIDEN_WARP = 10, WIDEN_WARPS = 2;
constexpr float P_SCALE = 256.f, MIN_LOG2_VSCALE = -64.f;
constexpr int MOST_ODD = 8;
constexpr int AT_O = 2 * KEYS; /* tensor memory: S at columns 0 and 64, O at 128 */

template <bool E4M3> struct Shape {
    static constexpr int THREADS = 32 * (E4M3 ? WIDEN_WARP + WIDEN_WARPS : WIDEN_WARP), BOUND = att::BOUND; /* 80 registers a thread: see there */
    static constexpr int Q_BYTES = 2 * ROWS * 128, K_BYTES = 2 * KEYS * 128, V_BYTES = K_BYTES;
    static constexpr int STAGES = E4M3 ? 1 : 2, RAW_STAGES = E4M3 ? 2 : 0;
    static constexpr int AT_K = Q_BYTES, AT_V = AT_K + STAGES * K_BYTES, AT_RAW = AT_V + STAGES * V_BYTES, AT_SCALE = AT_RAW + RAW_STAGES * PAGE_BYTES;
    static constexpr int SCALE_FLOATS = 3 * KEYS, AT_FACTOR = AT_SCALE + (E4M3 ? 2 * SCALE_FLOATS * 4 : 0), AT_STATE = AT_FACTOR + (E4M3 ? ROWS * 4 : 0);
    static constexpr int AT_BARS = AT_STATE + ROWS * 8, SMEM = 1024 + AT_BARS + 512;
    static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two blocks per SM");
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
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

template <bool E4M3> __global__ void __launch_bounds__(Shape<E4M3>::BOUND, 2) k_paged_tiles(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv,
                                                                                          const PagedArgs args) {
    using S = Shape<E4M3>;
    constexpr int STAGES = S::STAGES;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t *raw = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const ncb_paged &a = args.p;
    const uint32_t base = smem_u32(raw), bars = base + S::AT_BARS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(raw + S::AT_BARS + 256);
    volatile int *failed = reinterpret_cast<volatile int *>(raw + S::AT_BARS + 264);
    volatile int *odd_of = failed + 1; /* the b-th page that some row's border crosses has b + 1 at b % MOST_ODD if a value is not finite */
    volatile int *times = odd_of + MOST_ODD; /* how often a quarter's first warp has multiplied rows */
    /* the k-th page of the block uses entry k % 2 of each */
    auto k_full = [&](int k) { return bars + 8u * (k & 1); };
    auto v_full = [&](int k) { return bars + 16u + 8u * (k & 1); };
    auto s_full = [&](int k) { return bars + 32u + 8u * (k & 1); };
    auto p_ready = [&](int k) { return bars + 48u + 8u * (k & 1); };
    auto pv_done = [&](int k) { return bars + 64u + 8u * (k & 1); };
    auto raw_full = [&](int k) { return bars + 80u + 8u * (k & 1); };
    auto raw_free = [&](int k) { return bars + 96u + 8u * (k & 1); };
    const uint32_t q_full = bars + 112u, q_ready = bars + 120u, q_known = bars + 128u, looked = bars + 136u, o_free = bars + 144u, q_free = bars + 152u;
    auto stored = [&](int quarter) { return bars + 160u + 8u * quarter; };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(k_full(s), E4M3 ? WIDEN_WARPS : 1);
            mbar_init(v_full(s), E4M3 ? WIDEN_WARPS : 1);
            mbar_init(s_full(s), 1);
            mbar_init(p_ready(s), TILE_WARPS);
            mbar_init(pv_done(s), 1);
            mbar_init(raw_full(s), 1);
            mbar_init(raw_free(s), WIDEN_WARPS);
        }
        mbar_init(q_full, 1);
        mbar_init(q_ready, WIDEN_WARPS);
        mbar_init(q_known, TILE_WARPS);
        mbar_init(looked, TILE_WARPS);
        mbar_init(o_free, TILE_WARPS);
        mbar_init(q_free, 1);
        for (int quarter = 0; quarter < 4; quarter++) mbar_init(stored(quarter), 1);
        *failed = 0;
        for (int i = 0; i < MOST_ODD; i++) odd_of[i] = 0;
        for (int i = 0; i < 4; i++) times[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    /* The block's pieces: where tiles are whole, one owner, the longest first. What a piece is is read from the schedule again where it is needed: registers. */
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
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    att::fence_before();
    __syncthreads();
    att::fence_after();
    const uint32_t tmem = *tmem_slot;
    auto wait = [&](uint32_t bar, int use) { /* one thread */
        if (att::mbar_test(bar, use & 1)) return true;
        if (!*failed && mbar_wait(bar, use & 1)) return true;
        flag(a.status, NCB_DEV_WAIT_TIMEOUT);
        *failed = 1;
        return false;
    };
    auto wait_all = [&](uint32_t bar, int use) { return (bool)__all_sync(0xffffffffu, wait(bar, use)); }; /* a warp */
    auto load_piece = [&] {
        const int *w = a.work + class_at(args.caps, 1);
        if (!whole) return reinterpret_cast<const Piece *>(w + pieces_at(args.caps.tile))[piece];
        const Owner o = reinterpret_cast<const Owner *>(w + HEADER_WORDS)[piece];
        return Piece{o.request, o.row, o.rows, o.pos, o.page0, o.pages, (int)blockIdx.x % a.Hkv, -1};
    };
    auto begin_of = [&](int pos) { return a.window > 0 ? max(0, pos + 1 - a.window) : 0; };
    auto borders_of = [&](const Piece &e, int &lo, int &hi) { /* the border of some row's range lies in the pages before lo and in those from hi on */
        lo = (begin_of(e.pos + e.rows - 1) - e.page0 * KEYS + KEYS - 1) / KEYS, hi = (e.pos + 1) / KEYS - e.page0;
    };
    bool ok = true;
    int k = 0, q = 0, borders = 0; /* pages, pieces with pages, crossed pages before this piece */

    if (warp == COPY_WARP) {
        if (lane == 0) {
            const uint64_t keep = policy_evict_last();
            int v = 0;
            for (; ok && piece < pieces; piece++) {
                const Piece e = load_piece();
                if (e.pages == 0) continue;
                const int *table = a.table + (size_t)e.request * a.width + e.page0;
                int page = table[0];
                /* the products of the piece before have read its queries, and (E4M3) the softmax their factors */
                if (q > 0 && !((ok = wait(q_free, q - 1) && (!E4M3 || wait(q_known, q - 1))))) break;
                const int group = a.Hq / a.Hkv;
                mbar_expect_tx(q_full, 2 * (ROWS / group * group) * 128); /* a box is whole, whatever the tile uses of it */
                for (int j = 0; j < 2; j++) tma_load_3d(base + j * ROWS * 128, &map_q, 64 * j, e.head * group, e.row, q_full);
                q++;
                for (int i = 0; i < e.pages; i++) {
                    const int next = i + 1 < e.pages ? table[i + 1] : 0;
                    const bool in = (unsigned)page < (unsigned)a.n_pages;
                    if (!in) flag(a.status, NCB_DEV_BAD_PAGE);
                    if (E4M3) {
                        if (k >= 2 && !(ok = wait(raw_free(k), (k >> 1) - 1))) break;
                        mbar_expect_tx(raw_full(k), PAGE_BYTES); /* outside the pool: page 0, masked and widened to zeros */
                        bulk_load(base + S::AT_RAW + (k & 1) * PAGE_BYTES, (const uint8_t *)a.pool + ((size_t)(in ? page : 0) * a.Hkv + e.head) * PAGE_BYTES, PAGE_BYTES, raw_full(k));
                        k++;
                    } else { /* outside the pool: a box behind its end, zeros */
                        const int row = in ? (page * a.Hkv + e.head) * 2 * KEYS : a.n_pages * a.Hkv * 2 * KEYS, st = k & 1;
                        if (k >= 2 && !(ok = wait(s_full(k), (k >> 1) - 1))) break;
                        mbar_expect_tx(k_full(k), S::K_BYTES);
                        for (int j = 0; j < 2; j++) tma_load(base + S::AT_K + st * S::K_BYTES + j * KEYS * 128, &map_kv, 64 * j, row, k_full(k), keep);
                        k++;
                        if (v >= 2 && !(ok = wait(pv_done(v), (v >> 1) - 1))) break;
                        mbar_expect_tx(v_full(v), S::V_BYTES);
                        for (int j = 0; j < 2; j++) tma_load(base + S::AT_V + st * S::V_BYTES + j * KEYS * 128, &map_kv, 64 * j, row + KEYS, v_full(v), keep);
                        v++;
                    }
                    page = next;
                }
            }
            if (*failed) { /* the block must not leave under copies still in flight */
                if (q > 0) mbar_wait(q_full, (q - 1) & 1);
                for (int i = max(0, k - 2); i < k; i++) mbar_wait(E4M3 ? raw_full(i) : k_full(i), i >> 1 & 1);
                for (int i = max(0, v - 2); i < v; i++) mbar_wait(v_full(i), i >> 1 & 1);
            }
        }
    } else if (warp == MMA_WARP) { /* the warp goes through the loop together (elect_one) */
        constexpr uint32_t F32 = 1u << 4, BF16_AB = E4M3 ? 0u : (1u << 7) | (1u << 10), M = (uint32_t)(ROWS >> 4) << 24;
        constexpr uint32_t score = F32 | BF16_AB | M | ((uint32_t)(KEYS >> 3) << 17);
        constexpr uint32_t value = F32 | BF16_AB | M | ((uint32_t)(HEAD_DIM >> 3) << 17) | (E4M3 ? 0u : 1u << 16);
        const uint32_t t = __shfl_sync(0xffffffffu, tmem, 0), b = __shfl_sync(0xffffffffu, base, 0);
        for (; ok && piece < pieces; piece++) {
            const Piece e = load_piece();
            if (e.pages == 0) continue;
            auto scores = [&](int ki, bool last) {
                if (ki >= 2 && !wait_all(pv_done(ki), (ki - 2) >> 1)) return false; /* the buffer's probabilities have been used */
                if (!wait_all(k_full(ki), ki >> 1)) return false;
                att::fence_after();
                const uint32_t ks = b + S::AT_K + ki % STAGES * S::K_BYTES, d = t + (ki & 1) * KEYS;
                if (elect_one()) {
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int h = 0; h < 4; h++)
                            umma_bf16(d, umma_desc(b + j * ROWS * 128 + h * 32), umma_desc(ks + j * KEYS * 128 + h * 32), score, (j | h) != 0);
                    umma_commit(s_full(ki));
                    if (last) umma_commit(q_free);
                }
                __syncwarp();
                return true;
            };
            int lo, hi;
            borders_of(e, lo, hi);
            ok = wait_all(E4M3 ? q_ready : q_full, q) && scores(k, e.pages == 1);
            for (int i = 0; ok && i < e.pages; i++, k++) {
                ok = (i + 1 == e.pages || scores(k + 1, i + 2 == e.pages)) && wait_all(v_full(k), k >> 1) && wait_all(p_ready(k), k >> 1) && (i > 0 || q == 0 || wait_all(o_free, q - 1));
                if (!ok) break;
                att::fence_after();
                const uint32_t vs = b + S::AT_V + k % STAGES * S::V_BYTES, p = t + (k & 1) * KEYS;
                bool by_mma = true;
                if (i < lo || i >= hi) by_mma = odd_of[borders % MOST_ODD] != borders + 1, borders++;
                if (elect_one()) {
                    if (by_mma) {
#pragma unroll
                        for (int h = 0; h < KEYS / 16; h++) /* 16 keys: 8 columns of packed probabilities */
                            att::umma_from_tmem(t + AT_O, p + h * 8, E4M3 ? umma_desc(vs + h * 32) : att::desc_by_rows(vs + h * 2048, KEYS * 128), value, (i | h) != 0);
                    }
                    umma_commit(pv_done(k));
                }
                __syncwarp();
            }
            q++;
        }
    } else if (warp >= WIDEN_WARP) {
        if (E4M3) {
            constexpr int T = 32 * WIDEN_WARPS, ROUNDS = 512 / T;
            const int t = tid - 32 * WIDEN_WARP;
            for (; ok && piece < pieces; piece++) {
                const Piece e = load_piece();
                if (e.pages == 0) continue;
                const int *table = a.table + (size_t)e.request * a.width + e.page0;
                int page_at = table[0];
                if (!(ok = wait_all(q_full, q))) break;
                for (int r = t; r < ROWS; r += T) reinterpret_cast<float *>(raw + S::AT_FACTOR)[r] = query_row_to_f16(raw, r);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(q_ready);
                q++;
                for (int i = 0; ok && i < e.pages; i++, k++) {
                    const uint8_t *page = raw + S::AT_RAW + (k & 1) * PAGE_BYTES;
                    const bool in = (unsigned)page_at < (unsigned)a.n_pages;
                    page_at = i + 1 < e.pages ? table[i + 1] : 0;
                    ok = wait_all(raw_full(k), k >> 1);
                    if (!ok) break;
                    if (k >= 1 && !(ok = wait_all(s_full(k - 1), (k - 1) >> 1))) break; /* the scores before have read the keys' place */
                    { /* 16 codes -> 32 bytes: two chunks of a swizzled row */
                        const int j0 = t >> 3, c = t & 7;
                        uint8_t *keys = raw + S::AT_K + (c >> 2) * KEYS * 128 + j0 * 128;
                        const uint32_t at0 = ((2 * c & 7) ^ (j0 & 7)) << 4;
#pragma unroll
                        for (int half = 0; half < ROUNDS; half += 4) {
                            uint4 in4[4];
#pragma unroll
                            for (int y = 0; y < 4; y++) in4[y] = *reinterpret_cast<const uint4 *>(page + page_k_chunk(j0 + T / 8 * (half + y), c));
#pragma unroll
                            for (int y = 0; y < 4; y++) {
                                uint4 w[2];
                                widen_e4m3x4(in4[y].x, w[0].x, w[0].y), widen_e4m3x4(in4[y].y, w[0].z, w[0].w);
                                widen_e4m3x4(in4[y].z, w[1].x, w[1].y), widen_e4m3x4(in4[y].w, w[1].z, w[1].w);
                                uint8_t *row = keys + T / 8 * (half + y) * 128;
                                *reinterpret_cast<uint4 *>(row + at0) = w[0];
                                *reinterpret_cast<uint4 *>(row + (at0 ^ 16)) = w[1];
                            }
                        }
                    }
                    if (k >= 2 && !(ok = wait_all(pv_done(k), (k - 2) >> 1))) break; /* nobody reads these scales any more */
                    float *scales = reinterpret_cast<float *>(raw + S::AT_SCALE) + (k & 1) * S::SCALE_FLOATS;
                    const float vs = in ? reinterpret_cast<const float *>(page + PAGE_VS)[t] : 0.f;
                    scales[t] = in ? reinterpret_cast<const float *>(page + PAGE_KS)[t] : 0.f;
                    scales[KEYS + t] = fmaxf(log2_of(vs), MIN_LOG2_VSCALE);
                    scales[2 * KEYS + t] = vs * P_SCALE;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) arrive(k_full(k));
                    /* 16 positions of a dimension; those past the last row may hold anything: zeros */
                    const int used = in ? e.pos + e.rows - (e.page0 + i) * KEYS : 0;
                    if (k >= 1 && !(ok = wait_all(pv_done(k - 1), (k - 1) >> 1))) break; /* the values' place is free */
                    uint8_t *values = raw + S::AT_V + t * 128;
#pragma unroll
                    for (int half = 0; half < ROUNDS; half += 4) {
                        uint4 in4[4];
#pragma unroll
                        for (int y = 0; y < 4; y++) in4[y] = *reinterpret_cast<const uint4 *>(page + PAGE_V + (half + y) / 2 * 2048 + (t + T * (y & 1)) * 16);
                        if (used < KEYS) {
#pragma unroll
                            for (int y = 0; y < 4; y++)
#pragma unroll
                                for (int w = 0; w < 4; w++) {
                                    const int on = used - 16 * ((half + y) / 2) - 4 * w;
                                    (&in4[y].x)[w] = on >= 4 ? (&in4[y].x)[w] : on <= 0 ? 0u : (&in4[y].x)[w] & ((1u << (8 * on)) - 1u);
                                }
                        }
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            uint4 w[2];
                            widen_e4m3x4(in4[y].x, w[0].x, w[0].y), widen_e4m3x4(in4[y].y, w[0].z, w[0].w);
                            widen_e4m3x4(in4[y].z, w[1].x, w[1].y), widen_e4m3x4(in4[y].w, w[1].z, w[1].w);
                            uint8_t *row = values + T * (y & 1) * 128;
                            const uint32_t at = (((half + y) & 6) ^ (t & 7)) << 4; /* chunk 2 (y / 2) */
                            *reinterpret_cast<uint4 *>(row + at) = w[0];
                            *reinterpret_cast<uint4 *>(row + (at ^ 16)) = w[1];
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) arrive(v_full(k)), arrive(raw_free(k));
                }
            }
        }
    } else { /* softmax: a warp has 16 slots (two warps share a quarter of the lanes), a thread two of them */
        const int quarter = warp & 3, share = warp >> 2, first = quarter * 32 + share * 16, g = lane >> 2, t2 = (lane & 3) * 2;
        const uint32_t lanes = (uint32_t)first << 16, o_mine = tmem + AT_O + lanes, of_quarter = (uint32_t)(quarter * 32) << 16;
        for (; ok && piece < pieces; piece++) {
            const Piece e = load_piece();
            const int G = a.Hq / a.Hkv, slots = e.rows * G;
            if (e.pages == 0) { /* rows that are not served */
                for (int i = tid; i < slots * (HEAD_DIM / 8); i += 32 * TILE_WARPS) {
                    const int slot = i / (HEAD_DIM / 8);
                    *reinterpret_cast<uint4 *>((bf16 *)a.out + (size_t)(e.row + slot / G) * a.ldo + (size_t)(e.head * G + slot % G) * HEAD_DIM + i % (HEAD_DIM / 8) * 8) = make_uint4(0u, 0u, 0u, 0u);
                }
                continue;
            }
            float factor[2] = {args.scale_log2, args.scale_log2};
            if (E4M3) {
                if (!(ok = wait_all(q_ready, q))) break;
#pragma unroll
                for (int r = 0; r < 2; r++) factor[r] *= reinterpret_cast<const float *>(raw + S::AT_FACTOR)[first + g + 8 * r];
                __syncwarp();
                if (lane == 0) arrive(q_known);
                q++;
            }
            const int table = e.request * a.width + e.page0, pages = e.pages; /* requests * width is below 2^30 */
            auto last_of = [&](const Piece &e, int slot) { return e.pos + min(slot, e.rows * G - 1) / G; }; /* the last position that a slot sees */
            /* pages before lo and from hi on are crossed by the border of some row; those before my_lo and from my_hi on by one of this warp's. The loop keeps
             * little: what only such pages need is read from the schedule again there. */
            int lo, hi;
            borders_of(e, lo, hi);
            const int my_lo = (begin_of(last_of(e, first + 15)) - e.page0 * KEYS + KEYS - 1) / KEYS, my_hi = (last_of(e, first) + 1) / KEYS - e.page0;
            const bool idle = first >= slots; /* a warp without a slot only keeps the others company */
            const uint64_t factor2[2] = {att::pair_of(factor[0], factor[0]), att::pair_of(factor[1], factor[1])};
            float m[2] = {-INFINITY, -INFINITY};
            uint64_t sums[2] = {0, 0};
            bool pending = true; /* some row of the warp may have had no finite score yet */
            int page = a.table[table];
            for (int i = 0; i < pages; i++, k++) {
                const bool in = (unsigned)page < (unsigned)a.n_pages;
                page = i + 1 < pages ? a.table[table + i + 1] : 0;
                ok = wait_all(s_full(k), k >> 1);
                if (ok && E4M3) ok = wait_all(k_full(k), k >> 1); /* the scales were stored before it */
                if (!ok) break;
                att::fence_after();
                const uint32_t s_mine = tmem + (k & 1) * KEYS + lanes;
                const float *scales = reinterpret_cast<const float *>(raw + S::AT_SCALE) + (k & 1) * S::SCALE_FLOATS + t2;
                auto scale_at = [&](int j, int which) { return *reinterpret_cast<const uint64_t *>(scales + which * KEYS + j * 8); }; /* of 8 keys from 8 j */
                const bool border = i < lo || i >= hi;
                float s[32]; /* [8 keys][row][t2, t2 + 1] */
                float reference[2] = {0.f, 0.f};
                if (!idle) {
                    {
                        uint32_t bits[32];
                        att::tmem_rows64(s_mine, bits);
#pragma unroll
                        for (int j = 0; j < 32; j++) s[j] = __uint_as_float(bits[j]);
                    }
                    if (E4M3) {
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const uint64_t f = scale_at(j, 0);
                            att::mul2(s[4 * j], s[4 * j + 1], att::pair_of(s[4 * j], s[4 * j + 1]), f);
                            att::mul2(s[4 * j + 2], s[4 * j + 3], att::pair_of(s[4 * j + 2], s[4 * j + 3]), f);
                        }
                    }
                    if (i < my_lo || i >= my_hi || !in) { /* the border of some row crosses this warp's part of the page */
                        const Piece e = load_piece();
                        const int p0 = (e.page0 + i) * KEYS;
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            const int last = last_of(e, first + g + 8 * r), to = in ? last - p0 : -1, from = begin_of(last) - p0; /* in the page */
#pragma unroll
                            for (int j = 0; j < 16; j++) {
                                const int key = j / 2 * 8 + t2 + (j & 1);
                                float &y = s[j / 2 * 4 + 2 * r + (j & 1)];
                                y = key > to || key < from ? -INFINITY : y;
                            }
                        }
                    }
                    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < 8; j++)
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            float y = s[4 * j + 2 * r], z = s[4 * j + 2 * r + 1];
                            if (E4M3) att::fma2(y, z, att::pair_of(y, z), factor2[r], scale_at(j, 1)); /* the probabilities carry the value's scale */
                            best[r] = att::max3(best[r], y, z);
                        }
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        best[r] = fmaxf(best[r], __shfl_xor_sync(0xffffffffu, best[r], 1));
                        best[r] = fmaxf(best[r], __shfl_xor_sync(0xffffffffu, best[r], 2));
                        if (!E4M3) best[r] *= factor[r];
                    }
                    if (i == 0) {
                        m[0] = best[0], m[1] = best[1];
                    } else if (__any_sync(0xffffffffu, best[0] > m[0] + att::RESCALE_LOG2 || best[1] > m[1] + att::RESCALE_LOG2)) {
                        ok = wait_all(pv_done(k - 1), (k - 1) >> 1); /* O is complete up to the page before */
                        if (!ok) break;
                        att::fence_after();
                        float f[2];
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            const bool grown = best[r] > m[r] + att::RESCALE_LOG2;
                            f[r] = grown ? (m[r] == -INFINITY ? 0.f : ex2(m[r] - best[r])) : 1.f;
                            m[r] = grown ? best[r] : m[r];
                            sums[r] = att::mul2(sums[r], att::pair_of(f[r], f[r]));
                        }
#pragma unroll 1
                        for (int d = 0; d < HEAD_DIM / 32; d++) {
                            uint32_t y[16];
                            att::tmem_rows32(o_mine + d * 32, y);
#pragma unroll
                            for (int j = 0; j < 16; j++) y[j] = __float_as_uint(__uint_as_float(y[j]) * f[j >> 1 & 1]);
                            att::tmem_put_rows32(o_mine + d * 32, y);
                        }
                    }
                    reference[0] = m[0], reference[1] = m[1];
                    if (pending) {
                        const bool none[2] = {m[0] == -INFINITY, m[1] == -INFINITY};
                        pending = __any_sync(0xffffffffu, none[0] || none[1]);
                        reference[0] = none[0] ? 0.f : m[0], reference[1] = none[1] ? 0.f : m[1]; /* their scores are -infinity or NaN: nothing, or NaN */
                    }
                }
                if (border) {
                    ok = wait_all(v_full(k), k >> 1);
                    if (!ok) break;
                    uint8_t *v = raw + S::AT_V + k % STAGES * S::V_BYTES;
                    const Piece e = load_piece();
                    const int used = E4M3 ? KEYS : e.pos + e.rows - (e.page0 + i) * KEYS; /* positions past the last row may hold anything: zeros (E4M3: they are) */
                    bool strange = E4M3 && tid < KEYS && !isfinite((scales - t2)[2 * KEYS + tid]);
#pragma unroll 1
                    for (int y = tid; y < 2 * KEYS * 8; y += 32 * TILE_WARPS) {
                        uint4 *chunk = reinterpret_cast<uint4 *>(v) + y;
                        if (E4M3 || y / 8 % KEYS < used) strange |= att::not_finite8<E4M3>(*chunk);
                        else *chunk = make_uint4(0u, 0u, 0u, 0u);
                    }
                    if (!E4M3) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    strange = __any_sync(0xffffffffu, strange);
                    if (lane == 0) {
                        if (strange) odd_of[borders % MOST_ODD] = borders + 1;
                        arrive(looked);
                    }
                }
                if (!idle) {
                    const uint64_t minus[2] = {att::pair_of(-reference[0], -reference[0]), att::pair_of(-reference[1], -reference[1])};
#pragma unroll
                    for (int h = 0; h < 2; h++) { /* 32 keys: 16 packed columns */
                        uint32_t packed[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const int r = j & 1, at = 16 * h + 2 * j;
                            float y, z;
                            att::fma2(y, z, att::pair_of(s[at], s[at + 1]), factor2[r], minus[r]);
                            y = ex2(y), z = ex2(z);
                            const uint64_t yz = att::pair_of(y, z);
                            sums[r] = att::add2(sums[r], yz);
                            if (E4M3) {
                                att::mul2(y, z, yz, scale_at(4 * h + j / 2, 2));
                                packed[j] = f16_pair(y, z);
                            } else {
                                const __nv_bfloat162 w = __floats2bfloat162_rn(y, z);
                                packed[j] = *reinterpret_cast<const uint32_t *>(&w);
                            }
                        }
                        att::tmem_put_pairs16(s_mine + 16 * h, packed);
                    }
                    att::tmem_wait_store();
                }
                att::fence_before();
                __syncwarp();
                if (border) {
                    ok = wait_all(looked, borders);
                    if (!ok) break;
                    if (odd_of[borders % MOST_ODD] == borders + 1) { /* the quarter's first warp, a row per thread */
                        if (share == 1) {
                            if (lane == 0) arrive(stored(quarter));
                        } else {
                            ok = wait_all(stored(quarter), times[quarter]) && (i == 0 || wait_all(pv_done(k - 1), (k - 1) >> 1)); /* O is complete up to the page before */
                            if (!ok) break;
                            att::fence_after();
                            const Piece e = load_piece();
                            const int mine = last_of(e, quarter * 32 + lane), p0 = (e.page0 + i) * KEYS;
                            __syncwarp();
                            if (lane == 0) times[quarter] = times[quarter] + 1;
                            multiply_seen<E4M3>(raw + S::AT_V + k % STAGES * S::V_BYTES, tmem + (k & 1) * KEYS + of_quarter, tmem + AT_O + of_quarter, begin_of(mine) - p0, mine - p0 + 1, i == 0);
                            att::fence_before();
                            __syncwarp();
                        }
                    }
                    borders++;
                }
                if (lane == 0) arrive(p_ready(k));
            }
            ok = ok && wait_all(pv_done(k - 1), (k - 1) >> 1);
            if (!ok) break;
            float2 *state = reinterpret_cast<float2 *>(raw + S::AT_STATE);
#pragma unroll
            for (int r = 0; r < 2; r++) { /* each row's reference and sum */
                float l = __uint_as_float((uint32_t)sums[r]) + __uint_as_float((uint32_t)(sums[r] >> 32));
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                if (t2 == 0) state[first + g + 8 * r] = make_float2(m[r], l);
            }
            asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); /* the two warps of the quarter */
            { /* a thread has a row, its quarter's two warps every other 32 columns */
                const Piece e = load_piece();
                const int row = quarter * 32 + lane;
                const float2 ml = state[row];
                const bool on = row < slots;
                const float inv = ml.y > 0.f || ml.y != ml.y ? __fdiv_rn(1.f, E4M3 ? ml.y * P_SCALE : ml.y) : 0.f;
                bf16 *out = (bf16 *)a.out + (size_t)(e.row + (on ? row / G : 0)) * a.ldo + (size_t)(e.head * G + (on ? row % G : 0)) * HEAD_DIM;
                float *part = (float *)a.workspace + parts_at(args.caps, 1) + ((size_t)max(e.part, 0) * args.caps.tile.slots + row) * PART;
                att::fence_after();
                if (on && e.part >= 0 && share == 0) part[0] = ml.x, part[1] = ml.y;
#pragma unroll 1
                for (int d = share; d < HEAD_DIM / 32; d += 2) {
                    float y[32];
                    tmem_load32(tmem + AT_O + of_quarter + d * 32, y);
                    if (!on) continue;
                    if (e.part < 0) {
                        att::store32(out + d * 32, y, [&](int) { return inv; });
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(part + 4 + d * 32 + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
                    }
                }
                att::fence_before();
                __syncwarp();
                if (lane == 0) arrive(o_free);
            }
        }
    }
    att::fence_before();
    __syncthreads();
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
}

} /* namespace tiles */
} /* namespace */
