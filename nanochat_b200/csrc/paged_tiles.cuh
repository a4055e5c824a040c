/*
 * k_paged_tiles: attention of a tile of at most 128 query slots (new rows of one request x the query heads of a key/value head) over a run of
 * the request's pages, on tcgen05. A page's 64 keys at a time, as attn_tiles.cuh has it: S = Q K^T (M 128, N 64) into tensor memory, softmax in fp32 by
 * eight warps, the probabilities back over their scores, O += P V from there; two S buffers, so that the next page's scores run under
 * this page's softmax, and two blocks per SM. What is different here:
 *   - the slots of a tile are packed by row and head, so that a chunk of few rows still fills the MMAs and a page is read
 *     once for all heads of its group; queries come as one 3-d box (64 columns, the group's heads, the tile's rows);
 *   - pages are found through the block table; a page outside the pool is read as zeros (a box outside the tensor) and masked;
 *   - runs of pages, windows: rows may see nothing of a page at either end of their range, or nothing at all of a run;
 *   - bf16 pages: a probability enters P V as one bf16 term, 2^-9 of it away at most, and the sum it is divided by is that of the rounded terms:
 *     the tensor cores would need 512 cycles a page in place of 256 for two terms;
 *   - e4m3 pages: two warps widen a page to f16 in shared memory (keys in the form of a TMA box, values transposed as they lie), 500 issue slots a
 *     page, in place of a launch that widens a request's pages into a workspace of twice the pool's size. Queries are made f16 once per tile,
 *     each row times a power of two.
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

constexpr int ROWS = att::ROWS, KEYS = PAGE_TOKENS, SOFTMAX_WARPS = 8, COPY_WARP = 8, MMA_WARP = 9, WIDEN_WARP = 10, WIDEN_WARPS = 2;
constexpr int THREADS = 32 * (WIDEN_WARP + WIDEN_WARPS), BLOCKS = 2;
constexpr float P_SCALE = 256.f, MIN_LOG2_VSCALE = -64.f;
constexpr int MOST_ODD = 8;

template <bool E4M3> struct Shape {
    static constexpr int Q_BYTES = 2 * ROWS * 128, K_BYTES = 2 * KEYS * 128, V_BYTES = K_BYTES;
    static constexpr int K_STAGES = E4M3 ? 1 : 2, V_STAGES = E4M3 ? 1 : 2, RAW_STAGES = E4M3 ? 2 : 0;
    static constexpr int AT_K = Q_BYTES, AT_V = AT_K + K_STAGES * K_BYTES, AT_RAW = AT_V + V_STAGES * V_BYTES, AT_SCALE = AT_RAW + RAW_STAGES * PAGE_BYTES;
    static constexpr int AT_FACTOR = AT_SCALE + (E4M3 ? 2 * 3 * KEYS * 4 : 0), AT_BARS = AT_FACTOR + (E4M3 ? ROWS * 4 : 0);
    static constexpr int SMEM = 1024 + AT_BARS + 512;
    static_assert(BLOCKS * (SMEM + 1024) <= 228 * 1024, "two blocks per SM");
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

template <bool E4M3> __global__ void __launch_bounds__(THREADS, BLOCKS) k_paged_tiles(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv,
                                                                                    const PagedArgs args) {
    using S = Shape<E4M3>;
    constexpr int VB = 2;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t *raw = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const ncb_paged &a = args.p;
    const uint32_t base = smem_u32(raw), bars = base + S::AT_BARS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(raw + S::AT_BARS + 256);
    volatile int *failed = reinterpret_cast<volatile int *>(raw + S::AT_BARS + 264);
    volatile int *odd = failed + 1; /* per page that some row's border crosses: a value is not finite */
    auto k_full = [&](int s) { return bars + 8u * s; };
    auto v_full = [&](int s) { return bars + 16u + 8u * s; };
    auto s_full = [&](int s) { return bars + 32u + 8u * s; };
    auto p_ready = [&](int s) { return bars + 48u + 8u * s; };
    auto pv_done = [&](int s) { return bars + 64u + 8u * s; };
    const uint32_t q_full = bars + 80u, looked = bars + 88u, q_ready = bars + 96u;
    auto stored = [&](int quarter) { return bars + 104u + 8u * quarter; };
    auto raw_full = [&](int s) { return bars + 136u + 8u * s; };
    auto raw_free = [&](int s) { return bars + 152u + 8u * s; };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(k_full(s), E4M3 ? WIDEN_WARPS : 1);
            mbar_init(v_full(s), E4M3 ? WIDEN_WARPS : 1);
            mbar_init(s_full(s), 1);
            mbar_init(p_ready(s), SOFTMAX_WARPS);
            mbar_init(pv_done(s), 1);
            mbar_init(raw_full(s), 1);
            mbar_init(raw_free(s), WIDEN_WARPS);
        }
        mbar_init(q_full, 1);
        mbar_init(q_ready, WIDEN_WARPS);
        mbar_init(looked, SOFTMAX_WARPS);
        for (int quarter = 0; quarter < 4; quarter++) mbar_init(stored(quarter), 1);
        *failed = 0;
        for (int i = 0; i < MOST_ODD; i++) odd[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int entry = blockIdx.x / a.Hkv, kvh = blockIdx.x % a.Hkv, G = a.Hq / a.Hkv;
    if (entry >= a.work[2]) return; /* before any tensor memory is taken */
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    att::fence_before();
    __syncthreads();
    att::fence_after();
    const uint32_t tmem = *tmem_slot, t_out = tmem + 2 * KEYS; /* S at 0 and 64, O at 128 */
    const Entry e = reinterpret_cast<const Entry *>(a.work + entries_at(args.caps, 1))[entry];
    const int n = e.page1 - e.page0, slots = e.rows * G;
    const int pos0 = a.lens[e.request] - a.served[e.request] + e.row0, last_pos = pos0 + e.rows - 1;
    const long long first_row = a.row_start[e.request] + e.row0;
    const int *table = a.table + (size_t)e.request * a.width + e.page0;
    auto begin_of = [&](int pos) { return a.window > 0 ? max(0, pos + 1 - a.window) : 0; };
    const int all_from = begin_of(last_pos);
    auto crossed = [&](int i) { /* the border of some row's range lies in page i of the run */
        const int p0 = (e.page0 + i) * KEYS;
        return p0 + KEYS - 1 > pos0 || p0 < all_from;
    };
    auto wait = [&](uint32_t bar, int use) { /* one thread */
        if (att::mbar_test(bar, use & 1)) return true;
        if (!*failed && mbar_wait(bar, use & 1)) return true;
        flag(a.status, NCB_DEV_WAIT_TIMEOUT);
        *failed = 1;
        return false;
    };
    auto wait_all = [&](uint32_t bar, int use) { return (bool)__all_sync(0xffffffffu, wait(bar, use)); }; /* a warp */

    if (warp == COPY_WARP) {
        if (lane == 0 && n > 0) {
            const uint64_t keep = policy_evict_last();
            const int q_rows = ROWS / G * G; /* a box is whole, whatever the tile uses of it */
            mbar_expect_tx(q_full, 2 * q_rows * 128);
            for (int j = 0; j < 2; j++) tma_load_3d(base + j * ROWS * 128, &map_q, 64 * j, kvh * G, (int)first_row, q_full);
            int sent = 0, v_sent = 0, page = table[0];
            for (int i = 0; i < n; i++) {
                const int next = i + 1 < n ? table[i + 1] : 0;
                const bool ok = (unsigned)page < (unsigned)a.n_pages;
                if (!ok) flag(a.status, NCB_DEV_BAD_PAGE);
                if (E4M3) {
                    const int st = i & 1;
                    if (i >= 2 && !wait(raw_free(st), (i >> 1) - 1)) break;
                    mbar_expect_tx(raw_full(st), PAGE_BYTES); /* outside the pool: page 0, masked below and widened to zeros */
                    bulk_load(base + S::AT_RAW + st * PAGE_BYTES, (const uint8_t *)a.pool + ((size_t)(ok ? page : 0) * a.Hkv + kvh) * PAGE_BYTES, PAGE_BYTES, raw_full(st));
                    sent++;
                } else {
                    const int row = ok ? (page * a.Hkv + kvh) * 2 * KEYS : a.n_pages * a.Hkv * 2 * KEYS;
                    const int st = i & 1, before = i - 2;
                    if (before >= 0 && !wait(s_full(st), before >> 1)) break;
                    mbar_expect_tx(k_full(st), S::K_BYTES);
                    for (int j = 0; j < 2; j++) tma_load(base + S::AT_K + st * S::K_BYTES + j * KEYS * 128, &map_kv, 64 * j, row, k_full(st), keep);
                    sent++;
                    if (before >= 0 && !wait(pv_done(st), before >> 1)) break;
                    mbar_expect_tx(v_full(st), S::V_BYTES);
                    for (int j = 0; j < 2; j++) tma_load(base + S::AT_V + st * S::V_BYTES + j * KEYS * 128, &map_kv, 64 * j, row + KEYS, v_full(st), keep);
                    v_sent++;
                }
                page = next;
            }
            if (*failed) { /* the block must not leave under copies still in flight */
                mbar_wait(q_full, 0);
                for (int i = max(0, sent - 2); i < sent; i++) mbar_wait(E4M3 ? raw_full(i & 1) : k_full(i & 1), (i >> 1) & 1);
                for (int i = max(0, v_sent - 2); i < v_sent; i++) mbar_wait(v_full(i & 1), (i >> 1) & 1);
            }
        }
    } else if (warp == MMA_WARP) {
        if (n > 0) { /* the warp goes through the loop together (elect_one) */
            constexpr uint32_t F32 = 1u << 4, BF16_AB = E4M3 ? 0u : (1u << 7) | (1u << 10), M = (uint32_t)(ROWS >> 4) << 24;
            constexpr uint32_t score = F32 | BF16_AB | M | ((uint32_t)(KEYS >> 3) << 17);
            constexpr uint32_t value = F32 | BF16_AB | M | ((uint32_t)(HEAD_DIM >> 3) << 17) | (E4M3 ? 0u : 1u << 16);
            const uint32_t t = __shfl_sync(0xffffffffu, tmem, 0), b = __shfl_sync(0xffffffffu, base, 0), o = t + 2 * KEYS;
            auto scores = [&](int i) {
                const int st = E4M3 ? 0 : i & 1;
                if (i >= 2 && !wait_all(pv_done(i & 1), (i - 2) >> 1)) return false; /* the buffer's probabilities have been used */
                if (!wait_all(k_full(i & 1), i >> 1)) return false;
                att::fence_after();
                const uint32_t ks = b + S::AT_K + st * S::K_BYTES, d = t + (i & 1) * KEYS;
                if (elect_one()) {
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            umma_bf16(d, umma_desc(b + j * ROWS * 128 + k * 32), umma_desc(ks + j * KEYS * 128 + k * 32), score, (j | k) != 0);
                    umma_commit(s_full(i & 1));
                }
                __syncwarp();
                return true;
            };
            bool ok = wait_all(E4M3 ? q_ready : q_full, 0) && scores(0);
            int borders = 0;
            for (int i = 0; ok && i < n; i++) {
                if (i + 1 < n && !scores(i + 1)) break;
                const int st = E4M3 ? 0 : i & 1;
                if (!wait_all(v_full(i & 1), i >> 1) || !wait_all(p_ready(i & 1), i >> 1)) break;
                att::fence_after();
                const uint32_t vs = b + S::AT_V + st * S::V_BYTES, p = t + (i & 1) * KEYS;
                const bool by_mma = !crossed(i) || !odd[borders++ % MOST_ODD];
                if (elect_one()) {
                    if (by_mma) {
#pragma unroll
                        for (int k = 0; k < KEYS / 16; k++) /* 16 keys: 8 columns of packed probabilities */
                            att::umma_from_tmem(o, p + k * 8, E4M3 ? umma_desc(vs + k * 32) : att::desc_by_rows(vs + k * 2048, KEYS * 128), value, (i | k) != 0);
                    }
                    umma_commit(pv_done(i & 1));
                }
                __syncwarp();
            }
        }
    } else if (warp >= WIDEN_WARP) {
        if (E4M3 && n > 0) {
            const int t = tid - 32 * WIDEN_WARP; /* 0 .. 63 */
            if (wait_all(q_full, 0)) {
                for (int r = t; r < ROWS; r += 64) reinterpret_cast<float *>(raw + S::AT_FACTOR)[r] = query_row_to_f16(raw, r);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(q_ready);
            }
            for (int i = 0; i < n; i++) {
                const int st = i & 1;
                const uint8_t *page = raw + S::AT_RAW + st * PAGE_BYTES;
                const bool in = (unsigned)table[i] < (unsigned)a.n_pages;
                if (!wait_all(raw_full(st), i >> 1)) break;
                if (i >= 1 && !wait_all(s_full((i - 1) & 1), (i - 1) >> 1)) break; /* the scores before have read the keys' stage */
                uint8_t *k = raw + S::AT_K;
#pragma unroll 4
                for (int x = 0; x < 8; x++) { /* 16 codes -> 32 bytes: two chunks of a swizzled row */
                    const int at = t + 64 * x, j = at >> 3, c = at & 7;
                    const uint4 in4 = *reinterpret_cast<const uint4 *>(page + page_k_chunk(j, c));
                    uint4 y[2];
                    widen_e4m3x4(in4.x, y[0].x, y[0].y), widen_e4m3x4(in4.y, y[0].z, y[0].w);
                    widen_e4m3x4(in4.z, y[1].x, y[1].y), widen_e4m3x4(in4.w, y[1].z, y[1].w);
                    uint8_t *row = k + (c >> 2) * KEYS * 128 + j * 128;
                    *reinterpret_cast<uint4 *>(row + (((2 * c & 7) ^ (j & 7)) << 4)) = y[0];
                    *reinterpret_cast<uint4 *>(row + (((2 * c + 1 & 7) ^ (j & 7)) << 4)) = y[1];
                }
                if (i >= 2 && !wait_all(pv_done(i & 1), (i - 2) >> 1)) break; /* nobody reads these scales any more */
                float *scales = reinterpret_cast<float *>(raw + S::AT_SCALE) + st * 3 * KEYS;
                const float vs = in ? reinterpret_cast<const float *>(page + PAGE_VS)[t] : 0.f;
                scales[t] = in ? reinterpret_cast<const float *>(page + PAGE_KS)[t] : 0.f;
                scales[KEYS + t] = fmaxf(log2_of(vs), MIN_LOG2_VSCALE);
                scales[2 * KEYS + t] = vs * P_SCALE;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(k_full(st));
                if (i >= 1 && !wait_all(pv_done((i - 1) & 1), (i - 1) >> 1)) break; /* the values' stage is free */
                uint8_t *v = raw + S::AT_V;
                const int used = in ? last_pos + 1 - (e.page0 + i) * KEYS : 0; /* positions past the last row may hold anything: zeros */
#pragma unroll 4
                for (int x = 0; x < 8; x++) { /* 16 positions of a dimension */
                    const int at = t + 64 * x, group = at >> 7, d = at & 127;
                    uint4 in4 = *reinterpret_cast<const uint4 *>(page + PAGE_V + group * 2048 + d * 16);
                    const int left = used - 16 * group;
                    if (left < 16) {
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            const int on = left - 4 * w;
                            (&in4.x)[w] = on >= 4 ? (&in4.x)[w] : on <= 0 ? 0u : (&in4.x)[w] & ((1u << (8 * on)) - 1u);
                        }
                    }
                    uint4 y[2];
                    widen_e4m3x4(in4.x, y[0].x, y[0].y), widen_e4m3x4(in4.y, y[0].z, y[0].w);
                    widen_e4m3x4(in4.z, y[1].x, y[1].y), widen_e4m3x4(in4.w, y[1].z, y[1].w);
                    uint8_t *row = v + d * 128;
                    *reinterpret_cast<uint4 *>(row + ((2 * group ^ d & 7) << 4)) = y[0];
                    *reinterpret_cast<uint4 *>(row + ((2 * group + 1 ^ d & 7) << 4)) = y[1];
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(v_full(st)), arrive(raw_free(st));
            }
        }
    } else if (n > 0) { /* softmax: a warp has 16 slots (two warps share a quarter of the lanes), a thread two of them */
        const int quarter = warp & 3, share = warp >> 2, first = quarter * 32 + share * 16, g = lane >> 2, t2 = (lane & 3) * 2;
        const int see0 = pos0 + min(first, slots - 1) / G; /* the first slot's position */
        int to[2], from[2];
        float factor[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            to[r] = pos0 + min(first + g + 8 * r, slots - 1) / G, from[r] = begin_of(to[r]);
            factor[r] = args.scale_log2;
        }
        const int from_last = begin_of(pos0 + min(first + 15, slots - 1) / G);
        const bool idle = first >= slots; /* a warp without a slot only keeps the others company */
        bool ok = true;
        if (E4M3) {
            ok = wait_all(q_ready, 0);
#pragma unroll
            for (int r = 0; r < 2; r++) factor[r] *= reinterpret_cast<const float *>(raw + S::AT_FACTOR)[first + g + 8 * r];
        }
        const uint32_t lanes = (uint32_t)first << 16, o_mine = t_out + lanes, of_quarter = (uint32_t)(quarter * 32) << 16;
        const uint64_t factor2[2] = {att::pair_of(factor[0], factor[0]), att::pair_of(factor[1], factor[1])};
        float m[2] = {-INFINITY, -INFINITY};
        uint64_t sums[2] = {0, 0};
        int multiplied = 0, borders = 0;
        bool pending = true; /* some row of the warp may have had no finite score yet */
        int page = table[0];
        for (int i = 0; ok && i < n; i++) {
            const bool in = (unsigned)page < (unsigned)a.n_pages;
            page = i + 1 < n ? table[i + 1] : 0;
            ok = wait_all(s_full(i & 1), i >> 1);
            if (ok && E4M3) ok = wait_all(k_full(i & 1), i >> 1); /* the scales were stored before it */
            if (!ok) break;
            att::fence_after();
            const int p0 = (e.page0 + i) * KEYS, vst = E4M3 ? 0 : i & 1;
            const uint32_t s_mine = tmem + (i & 1) * KEYS + lanes;
            const float *scales = reinterpret_cast<const float *>(raw + S::AT_SCALE) + (i & 1) * 3 * KEYS + t2;
            auto scale_at = [&](int j, int which) { return *reinterpret_cast<const uint64_t *>(scales + which * KEYS + j * 8); }; /* of 8 keys from 8 j */
            const bool border = crossed(i);
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
                if (p0 + KEYS - 1 > see0 || p0 < from_last || !in) { /* the border of some row crosses this warp's part of the page */
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const int pos = p0 + j / 4 * 8 + t2 + (j & 1), r = j >> 1 & 1;
                        s[j] = pos > to[r] || pos < from[r] || !in ? -INFINITY : s[j];
                    }
                }
                float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        float x = s[4 * j + 2 * r], y = s[4 * j + 2 * r + 1];
                        if (E4M3) att::fma2(x, y, att::pair_of(x, y), factor2[r], scale_at(j, 1)); /* the probabilities carry the value's scale */
                        best[r] = att::max3(best[r], x, y);
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
                    ok = wait_all(pv_done((i - 1) & 1), (i - 1) >> 1); /* O is complete up to the page before */
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
                    for (int c = 0; c < VB * 2; c++) {
                        uint32_t o[16];
                        att::tmem_rows32(o_mine + c * 32, o);
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f[j >> 1 & 1]);
                        att::tmem_put_rows32(o_mine + c * 32, o);
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
                ok = wait_all(v_full(i & 1), i >> 1);
                if (!ok) break;
                uint8_t *v = raw + S::AT_V + vst * S::V_BYTES;
                const int used = E4M3 ? KEYS : last_pos + 1 - p0; /* positions past the last row may hold anything: zeros (E4M3: they are) */
                bool strange = E4M3 && tid < KEYS && !isfinite((scales - t2)[2 * KEYS + tid]);
#pragma unroll
                for (int c = tid; c < VB * KEYS * 8; c += 32 * SOFTMAX_WARPS) {
                    uint4 *chunk = reinterpret_cast<uint4 *>(v) + c;
                    if (E4M3 || c / 8 % KEYS < used) strange |= att::not_finite8<E4M3>(*chunk);
                    else *chunk = make_uint4(0u, 0u, 0u, 0u);
                }
                if (!E4M3) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                strange = __any_sync(0xffffffffu, strange);
                if (lane == 0) {
                    if (strange) odd[borders % MOST_ODD] = 1;
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
                        float x, y;
                        att::fma2(x, y, att::pair_of(s[at], s[at + 1]), factor2[r], minus[r]);
                        x = ex2(x), y = ex2(y);
                        if (E4M3) {
                            const uint64_t xy = att::pair_of(x, y);
                            sums[r] = att::add2(sums[r], xy);
                            att::mul2(x, y, xy, scale_at(4 * h + j / 2, 2));
                            packed[j] = f16_pair(x, y);
                        } else {
                            const __nv_bfloat162 z = __floats2bfloat162_rn(x, y);
                            packed[j] = *reinterpret_cast<const uint32_t *>(&z);
                            sums[r] = att::add2(sums[r], att::pair_of(__uint_as_float(packed[j] << 16), __uint_as_float(packed[j] & 0xffff0000u)));
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
                if (odd[borders % MOST_ODD]) { /* the quarter's first warp, a row per thread */
                    if (share == 1) {
                        if (lane == 0) arrive(stored(quarter));
                    } else {
                        ok = wait_all(stored(quarter), multiplied++) && (i == 0 || wait_all(pv_done((i - 1) & 1), (i - 1) >> 1)); /* O is complete up to the page before */
                        if (!ok) break;
                        att::fence_after();
                        const int mine = pos0 + min(quarter * 32 + lane, slots - 1) / G;
                        multiply_seen<E4M3>(raw + S::AT_V + vst * S::V_BYTES, tmem + (i & 1) * KEYS + of_quarter, t_out + of_quarter, begin_of(mine) - p0, mine - p0 + 1, i == 0);
                        att::fence_before();
                        __syncwarp();
                    }
                }
                borders++;
            }
            if (lane == 0) arrive(p_ready(i & 1));
        }
        ok = ok && wait_all(pv_done((n - 1) & 1), (n - 1) >> 1);
        /* each row's reference and sum, where the queries were (no product reads them any more) */
        float2 *state = reinterpret_cast<float2 *>(raw);
#pragma unroll
        for (int r = 0; r < 2; r++) {
            float l = __uint_as_float((uint32_t)sums[r]) + __uint_as_float((uint32_t)(sums[r] >> 32));
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (ok && t2 == 0) state[first + g + 8 * r] = make_float2(m[r], l);
        }
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); /* the two warps of the quarter */
        if (ok) { /* a thread has a row, its quarter's two warps every other 32 columns */
            const int row = quarter * 32 + lane;
            const float2 ml = state[row];
            const bool on = row < slots;
            const int head = kvh * G + (on ? row % G : 0);
            const long long out_row = first_row + (on ? row / G : 0);
            const float inv = ml.y > 0.f || ml.y != ml.y ? __fdiv_rn(1.f, E4M3 ? ml.y * P_SCALE : ml.y) : 0.f;
            float *part = (float *)a.workspace + parts_at(args.caps, a.Hkv, 1) + ((size_t)((long long)e.part * a.Hkv + kvh) * args.caps.tile.slots + row) * PART;
            att::fence_after();
            if (on && e.part >= 0 && share == 0) part[0] = ml.x, part[1] = ml.y;
#pragma unroll 1
            for (int c = share; c < VB * 2; c += 2) {
                float o[32];
                tmem_load32(t_out + of_quarter + c * 32, o);
                if (!on) continue;
                if (e.part < 0) {
                    att::store32((bf16 *)a.out + out_row * a.ldo + (size_t)head * HEAD_DIM + c * 32, o, [&](int) { return inv; });
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(part + 4 + c * 32 + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                }
            }
        }
    }
    if (n == 0) /* rows that were not served */
        for (int i = tid; i < slots * (HEAD_DIM / 8); i += blockDim.x) {
            const int slot = i / (HEAD_DIM / 8);
            *reinterpret_cast<uint4 *>((bf16 *)a.out + (first_row + slot / G) * a.ldo + (size_t)(kvh * G + slot % G) * HEAD_DIM + i % (HEAD_DIM / 8) * 8) = make_uint4(0u, 0u, 0u, 0u);
        }
    att::fence_before();
    __syncthreads();
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
}

} /* namespace tiles */
} /* namespace */
