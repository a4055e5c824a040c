/*
 * Attention of every request's new rows over its pages (page_plan.cu makes block tables and schedules, paged_append.cu fills the pages).
 * Replaces the reference's k_attn (model/kernels/decode.cu:567-675), which reads one slot's contiguous rows, for pools of pages,
 * grouped query heads, split lengths and several new rows per request.
 *
 * k_paged_small, for requests of at most 16 query slots (new rows x the heads of a key/value head's group): bound by the stream of pages. A block of
 * four warps (twelve: see the launch) walks over the pieces of its part of the line (paged.cuh); each warp fetches every fourth unit (an e4m3 page, half a bf16 page) into a place of its
 * own, consumes it and fetches its next: three blocks per SM keep twelve units of 16 KB in flight or in use, and no warp waits for another until the piece ends.
 * 64 requests of 8,191 positions, 32 heads over 8, e4m3: 167 us with the join, 6.6 TB/s; 45 of 130 to 16,384, 16 over 4, bf16: 58.5 us, 5.7 TB/s (device alone; 170 and 61 as calls). Requests of 17 to 32 slots
 * as two owners here in place of tiles: e4m3 41 us for 44, bf16 43 for 40; of 64 slots 75 for 59.
 * The CACHE is the A operand of both products (m16n8k16: 16 keys, or 16 dims of V^T), the slots its 8 columns (two tiles of them for more than 8), so
 * that few slots waste little; score accumulators become the B operand of V^T P by 8 x 8 transposes.
 *   - bf16 pages: a probability enters as two bf16 terms (hi + lo, 16 bits): one term would double the error of the bf16 output, and the
 *     stream of pages leaves the MMAs time;
 *   - e4m3 pages: bytes widened to f16 (exact) in registers, queries f16 after a power-of-two scale, the key's scale on the fp32 score, the value's folded
 *     into the f16 probability (11 bits), the running maximum that of score + log2(value scale), as in decode_attn.cu.
 * What a row does not see must not reach it, not even as zero times a NaN or an infinity: scores are masked by selects, and a unit that is not
 * seen whole by every slot has its values looked at; if one is not finite, its products are made row by row over the keys seen.
 *
 * k_paged_tiles (paged_tiles.cuh), for the others: tcgen05. k_paged_merge: the states of owners that were cut. A call launches the kernels that its sizes may need, and
 * which of them has something to do is the schedule's to say.
 * Waits are bounded: when one expires NCB_DEV_WAIT_TIMEOUT is flagged and the block leaves after its copies in flight.
 */
#include <atomic>

#include "paged_tiles.cuh"

namespace {

using namespace paged;

constexpr int FEW = 4, MANY = 12; /* warps of a block, of which three or one are on an SM */
constexpr float LOG2_E = 1.4426950408889634f;
constexpr float P_SCALE = 256.f; /* keeps small folded probabilities among f16's normal numbers; an exact power of two */
constexpr float MIN_LOG2_VSCALE = -64.f;
constexpr int BOX_ROWS = 32, BOX_BYTES = BOX_ROWS * 128;

/* What a warp fetches and consumes at a time: an e4m3 page, or half a bf16 page (four boxes of 32 rows x 64 columns, swizzled: keys' columns 0 .. 63
 * and 64 .. 127, then the values'). */
template <bool E4M3, int WARPS> struct Unit {
    static constexpr int KEYS = E4M3 ? PAGE_TOKENS : PAGE_TOKENS / 2, PER_PAGE = PAGE_TOKENS / KEYS;
    static constexpr int BYTES = E4M3 ? PAGE_BYTES : 4 * BOX_BYTES;
    static constexpr int BLOCKS = MANY / WARPS;
    static constexpr int SMEM = 1024 + WARPS * BYTES; /* 1024: swizzled boxes are aligned by hand */
    static_assert(BLOCKS * (SMEM + 2048) <= 228 * 1024, "blocks per SM");
    static_assert(SMALL_SLOTS * PART * 4 <= BYTES, "a warp's states lie where its unit was");
};

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool F16> __device__ __forceinline__ void mma16(float *d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t *b) {
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void ldmatrix4(uint32_t *r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t *r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
/* An 8 x 8 matrix of 16-bit values, row lane / 4 with columns 2 (lane % 4) and the next, to its transpose in the same form. */
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float quad_max(float v) { /* over lanes of the same lane / 4 */
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float column_max(float v) { /* over lanes of the same lane % 4 */
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
__device__ __forceinline__ void bulk_load_once(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy) : "memory");
}

/* Past L1, of what nobody writes while the kernel runs: free to move, unlike __ldcg, which cost the stream of pages 1 us of 60. (Not before the wait for the launches before:
 * the addresses come from the schedule, which is read behind it.) */
__device__ __forceinline__ uint2 two_words_of_l2(const bf16 *at) {
    uint2 x;
    asm("ld.global.cg.v2.u32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "l"(at));
    return x;
}
template <typename Word> __device__ __forceinline__ uint32_t word_of_l2(const Word *at) {
    uint32_t x;
    asm("ld.global.cg.u32 %0, [%1];" : "=r"(x) : "l"(at));
    return x;
}

/* What a state (m, l) counts relative to 2^top: nothing where it holds nothing. */
__device__ __forceinline__ float scale_of(float m, float l, float top) { return m == -INFINITY && l == l ? 0.f : ex2(m - top); }

/* Value `dim` of position j of a unit. */
template <bool E4M3> __device__ __forceinline__ float value_at(const uint8_t *unit, int j, int dim) {
    if (E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw(unit[page_v_byte(j, dim)], __NV_E4M3)));
    return __bfloat162float(*reinterpret_cast<const bf16 *>(unit + (2 + dim / 64) * BOX_BYTES + j * 128 + ((dim % 64 / 8 ^ j & 7) * 16) + dim % 8 * 2));
}

/* Whether some value of the 16 positions from `key` is infinite or NaN (a warp). */
template <bool E4M3> __device__ __forceinline__ bool strange_values(const uint8_t *unit, int key, int lane) {
    bool strange = false;
    if (E4M3) { /* 2,048 bytes, a position's codes at the same byte of 128 chunks; NaN is 0x7f with either sign */
        const uint4 *v = reinterpret_cast<const uint4 *>(unit + page_v_byte(key, 0));
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
            const uint4 x = v[lane + 32 * i];
#pragma unroll
            for (int e = 0; e < 4; e++) strange |= __vcmpeq4((&x.x)[e] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
        }
    } else {
        const uint4 *v = reinterpret_cast<const uint4 *>(unit + (2 + (lane & 1)) * BOX_BYTES + (key + (lane >> 1)) * 128); /* half a row a lane */
#pragma unroll 1
        for (int i = 0; i < 8; i++) {
            uint32_t acc = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"((&v[i].x)[e]), "r"(0u));
            strange |= (acc & 0x7fff7fffu) != 0;
        }
    }
    return __any_sync(0xffffffffu, strange);
}

template <bool E4M3, int NT, int WARPS> __global__ void __launch_bounds__(32 * WARPS, MANY / WARPS) k_paged_small(const __grid_constant__ CUtensorMap map, const PagedArgs args) {
    using U = Unit<E4M3, WARPS>;
    constexpr int TILES = U::KEYS / 16; /* of 16 keys */
    extern __shared__ __align__(128) uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[WARPS];
    __shared__ int failed;
    __shared__ float state_m[WARPS][8 * NT], state_l[WARPS][8 * NT];
    const ncb_paged &a = args.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t *smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const uint8_t *unit = smem + warp * U::BYTES;
    const uint32_t unit_u = smem_u32(unit), bar = smem_u32(bars + warp);
    if (tid == 0) {
        for (int w = 0; w < WARPS; w++) mbar_init(smem_u32(bars + w), 1);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    /* Behind the tile kernel of the same call there is nothing to wait for, since its blocks began after the launches before the call: these blocks fill SMs that its last ones
     * leave idle. (What they read was written before; it is read past L1, which need not have been emptied since.) They end after it, so that whoever waits for them
     * waits for both. */
    if (!args.caps.tiles) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int G = a.Hq / a.Hkv;
    const uint64_t once = policy_evict_first();
    uint32_t loads = 0; /* of this warp so far: the parity of its barrier */
    bool there = false; /* the unit in its place is in the pool */
    const Line line(args, 0);
    Start start = {(int)blockIdx.x / a.Hkv, (int)blockIdx.x % a.Hkv, 0, 0};
    long long left;
    const bool whole = WARPS > FEW || line.whole; /* one owner, to its end */
    if (whole) {
        left = WARPS > FEW || start.owner < line.n ? 1 << 30 : 0;
    } else {
        start = of_l2(line.starts + blockIdx.x);
        left = max(0ll, min(line.all() - blockIdx.x * line.share, line.share));
    }
    Walk walk(line.owners, line.n, line.overhead, start, (int)left, blockIdx.x);
    while (walk.next()) {
        if (WARPS > FEW && start.owner >= line.n) break; /* looked at only here: the owner's record comes beside the header */
        const Owner &e = walk.o;
        const int kvh = walk.head, page0 = e.page0 + walk.page0, part_at = walk.part;
        const int slots = e.rows * G, units = (walk.page1 - walk.page0) * U::PER_PAGE, first_pos = e.pos, last_pos = e.pos + e.rows - 1;
        const long long first_row = e.row;
        const int *table = a.table + (size_t)e.request * a.width + page0;
        auto begin_of = [&](int pos) { return a.window > 0 ? max(0, pos + 1 - a.window) : 0; }; /* the first position that the row at pos sees */
        /* The piece's unit i, of this page, into the warp's place; a page that is not in the pool is left out. */
        auto fetch = [&](int i, int page) {
            there = (unsigned)page < (unsigned)a.n_pages;
            if (lane != 0) return;
            if (!there) {
                flag(a.status, NCB_DEV_BAD_PAGE);
                att::arrive(bar);
                return;
            }
            mbar_expect_tx(bar, U::BYTES);
            if (E4M3) {
                bulk_load_once(unit_u, (const uint8_t *)a.pool + ((size_t)page * a.Hkv + kvh) * PAGE_BYTES, PAGE_BYTES, bar, once);
            } else {
                const int row = (page * a.Hkv + kvh) * 2 * PAGE_TOKENS + i % U::PER_PAGE * BOX_ROWS;
#pragma unroll
                for (int x = 0; x < 4; x++) tma_load(unit_u + x * BOX_BYTES, &map, 64 * (x & 1), row + (x >> 1) * PAGE_TOKENS, bar, once);
            }
        };
        if (warp < units) fetch(warp, (int)word_of_l2(table + warp / U::PER_PAGE));
        /* ---- queries: column n = lane / 4 of tile nt is slot 8 nt + n; k slots (2t, 2t+1), (2t+8, 2t+9) of step s are dims 16 s + 2 t .. and + 8, or (E4M3)
         * 16 s + 4 t .. + 3, as the cache bytes arrive ---- */
        uint32_t qb[NT][8][2];
        float factor[NT][2]; /* of the scores of slots 8 nt + 2 t and the next */
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int slot = 8 * nt + g;
            const bool on = slot < slots;
            const bf16 *src = (const bf16 *)a.q + (first_row + (on ? slot / G : 0)) * a.ldq + (size_t)(kvh * G + (on ? slot % G : 0)) * HEAD_DIM;
            float back = 1.f;
            if (E4M3) {
                float most = 0.f;
                uint2 u[8];
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    u[s] = on ? two_words_of_l2(src + 16 * s + 4 * t) : make_uint2(0u, 0u);
                    most = fmaxf(most, fmaxf(fmaxf(fabsf(__uint_as_float(u[s].x << 16)), fabsf(__uint_as_float(u[s].x & 0xffff0000u))),
                                             fmaxf(fabsf(__uint_as_float(u[s].y << 16)), fabsf(__uint_as_float(u[s].y & 0xffff0000u)))));
                }
                most = quad_max(most);
                /* the row's largest magnitude to [2^14, 2^15): what f16 then rounds or loses is below 2^-38 of it */
                const int expo = (int)((__float_as_uint(most) >> 23) & 0xffu) - 127, down = max(-100, min(expo - 14, 112));
                const float mul = __uint_as_float((uint32_t)(127 - down) << 23);
                back = __uint_as_float((uint32_t)(127 + down) << 23);
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    qb[nt][s][0] = pack_f16(__uint_as_float(u[s].x << 16) * mul, __uint_as_float(u[s].x & 0xffff0000u) * mul);
                    qb[nt][s][1] = pack_f16(__uint_as_float(u[s].y << 16) * mul, __uint_as_float(u[s].y & 0xffff0000u) * mul);
                }
            } else {
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    qb[nt][s][0] = on ? word_of_l2(src + 16 * s + 2 * t) : 0u;
                    qb[nt][s][1] = on ? word_of_l2(src + 16 * s + 8 + 2 * t) : 0u;
                }
            }
#pragma unroll
            for (int x = 0; x < 2; x++) factor[nt][x] = args.scale_log2 * (E4M3 ? __shfl_sync(0xffffffffu, back, (2 * t + x) * 4) : 1.f);
        }
        const int all_from = begin_of(last_pos), all_to = first_pos, any_from = begin_of(first_pos); /* what every slot sees; what some slot sees */
        float m[NT][2], l[NT][2], o[NT][8][4]; /* o: dims 16 d + lane / 4 (+ 8) of slots 2 t, 2 t + 1 */
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int x = 0; x < 2; x++) m[nt][x] = -INFINITY, l[nt][x] = 0.f;
#pragma unroll
            for (int d = 0; d < 8; d++)
#pragma unroll
                for (int x = 0; x < 4; x++) o[nt][d][x] = 0.f;
        }
        for (int i = warp; i < units; i += WARPS) {
            const int unit_pos = (page0 * U::PER_PAGE + i) * U::KEYS;
            const int next = i + WARPS < units ? (int)word_of_l2(table + (i + WARPS) / U::PER_PAGE) : 0;
            if (!__all_sync(0xffffffffu, mbar_wait(bar, loads++ & 1))) {
                if (lane == 0) flag(a.status, NCB_DEV_WAIT_TIMEOUT), failed = 1;
                mbar_wait(bar, loads - 1 & 1); /* nobody leaves under a copy */
                break;
            }
            if (there && unit_pos <= last_pos && unit_pos + U::KEYS > any_from) {
                /* ---- scores: tile k, element x: key row lane / 4 (x < 2) or 8 + lane / 4 of the tile, slots 2 t + x % 2. Rows are keys in order, or (E4M3) rows r and
                 * 8 + r keys 4 (r / 2) + r % 2 and 2 more, so that their transposes meet four consecutive bytes of V^T ---- */
                const int row[2] = {E4M3 ? 4 * (g >> 1) + (g & 1) : g, E4M3 ? 4 * (g >> 1) + (g & 1) + 2 : g + 8};
                float s[TILES][NT][4];
#pragma unroll
                for (int k = 0; k < TILES; k++) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int x = 0; x < 4; x++) s[k][nt][x] = 0.f;
                    const int mi = lane >> 3, r = lane & 7;
                    if (E4M3) { /* matrices: rows 0 .. 7, 8 .. 15 of 16 dims, then of the next 16 */
                        const int j = 16 * k + 4 * (r >> 1) + (r & 1) + 2 * (mi & 1);
                        const uint32_t at = unit_u + PAGE_K + j * HEAD_DIM, swz = (uint32_t)((j >> 2) & 7);
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            uint32_t w[4], f[4][2];
                            ldmatrix4(w, at + (((2 * c + (mi >> 1)) ^ swz) << 4));
#pragma unroll
                            for (int x = 0; x < 4; x++) widen_e4m3x4(w[x], f[x][0], f[x][1]);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                mma16<true>(s[k][nt], f[0][0], f[1][0], f[0][1], f[1][1], qb[nt][2 * c]);
                                mma16<true>(s[k][nt], f[2][0], f[3][0], f[2][1], f[3][1], qb[nt][2 * c + 1]);
                            }
                        }
                    } else { /* matrices: rows 0 .. 7, 8 .. 15 of 8 dims, then of the next 8 */
                        const int j = 16 * k + r + 8 * (mi & 1);
                        const uint32_t at = unit_u + j * 128;
#pragma unroll
                        for (int c = 0; c < 8; c++) {
                            uint32_t w[4];
                            ldmatrix4(w, at + (c >> 2) * BOX_BYTES + (((2 * (c & 3) + (mi >> 1)) ^ (j & 7)) << 4));
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma16<false>(s[k][nt], w[0], w[1], w[2], w[3], qb[nt][c]);
                        }
                    }
                }
                const bool masked = unit_pos < all_from || unit_pos + U::KEYS - 1 > all_to;
                float best[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) best[nt][0] = best[nt][1] = -INFINITY;
                float vs[TILES][2];
#pragma unroll
                for (int k = 0; k < TILES; k++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float ks = 1.f, lv = 0.f;
                        if (E4M3) {
                            ks = *reinterpret_cast<const float *>(unit + PAGE_KS + (16 * k + row[h]) * 4);
                            vs[k][h] = *reinterpret_cast<const float *>(unit + PAGE_VS + (16 * k + row[h]) * 4);
                            lv = fmaxf(lg2(vs[k][h]), MIN_LOG2_VSCALE);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int x = 0; x < 2; x++) {
                                float &y = s[k][nt][2 * h + x];
                                y *= E4M3 ? ks * factor[nt][x] : factor[nt][x];
                                if (masked) {
                                    const int pos = unit_pos + 16 * k + row[h], mine = first_pos + min(8 * nt + 2 * t + x, slots - 1) / G;
                                    if (pos > mine || pos < begin_of(mine)) y = -INFINITY;
                                }
                                best[nt][x] = fmaxf(best[nt][x], y + lv);
                            }
                    }
                bool moved = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        best[nt][x] = fmaxf(column_max(best[nt][x]), m[nt][x]);
                        moved |= best[nt][x] > m[nt][x];
                    }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float f[2];
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            f[x] = m[nt][x] == -INFINITY ? 0.f : ex2(m[nt][x] - best[nt][x]);
                            m[nt][x] = best[nt][x];
                            l[nt][x] *= f[x];
                        }
#pragma unroll
                        for (int d = 0; d < 8; d++) o[nt][d][0] *= f[0], o[nt][d][1] *= f[1], o[nt][d][2] *= f[0], o[nt][d][3] *= f[1];
                    }
                }
#pragma unroll
                for (int k = 0; k < TILES; k++) {
                    uint32_t p[E4M3 ? 1 : 2][NT][2]; /* the B operand of the values' product: hi and lo terms, or one f16 */
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            float w[2];
#pragma unroll
                            for (int x = 0; x < 2; x++) {
                                /* nothing counts yet where the maximum is -infinity; NaN scores stay NaN */
                                w[x] = ex2(s[k][nt][2 * h + x] - (m[nt][x] == -INFINITY ? 0.f : m[nt][x]));
                                l[nt][x] += w[x];
                                if (E4M3) w[x] = masked && s[k][nt][2 * h + x] == -INFINITY ? 0.f : w[x] * (vs[k][h] * P_SCALE);
                                s[k][nt][2 * h + x] = w[x];
                            }
                            if (E4M3) {
                                p[0][nt][h] = transposed(pack_f16(w[0], w[1]));
                            } else {
                                const uint32_t hi = pack_bf16(w[0], w[1]);
                                p[0][nt][h] = transposed(hi);
                                p[E4M3 ? 0 : 1][nt][h] = transposed(pack_bf16(w[0] - __uint_as_float(hi << 16), w[1] - __uint_as_float(hi & 0xffff0000u)));
                            }
                        }
                    if (masked && (unit_pos + 16 * k > last_pos || unit_pos + 16 * k + 15 < any_from)) continue; /* no slot sees any of it */
                    if (masked && strange_values<E4M3>(unit, 16 * k, lane)) { /* rare: key by key, for the slots that see it */
#pragma unroll 1
                        for (int j = 0; j < 16; j++) {
                            const int pos = unit_pos + 16 * k + j, h = E4M3 ? j >> 1 & 1 : j >> 3, from = E4M3 ? (j >> 2) * 2 + (j & 1) : j & 7;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                for (int x = 0; x < 2; x++) {
                                    const float w = __shfl_sync(0xffffffffu, h ? s[k][nt][2 + x] : s[k][nt][x], from * 4 + t);
                                    const int mine = first_pos + min(8 * nt + 2 * t + x, slots - 1) / G;
                                    if (pos > mine || pos < begin_of(mine)) continue;
#pragma unroll
                                    for (int d = 0; d < 8; d++) {
                                        o[nt][d][x] = fmaf(w, value_at<E4M3>(unit, 16 * k + j, 16 * d + g), o[nt][d][x]);
                                        o[nt][d][2 + x] = fmaf(w, value_at<E4M3>(unit, 16 * k + j, 16 * d + 8 + g), o[nt][d][2 + x]);
                                    }
                                }
                        }
                        continue;
                    }
                    /* ---- values: A = V^T, 16 dims by 16 keys ---- */
                    const int mi = lane >> 3, r = lane & 7;
                    if (E4M3) {
                        const uint32_t at = unit_u + page_v_byte(16 * k, 0) + lane * 16;
#pragma unroll
                        for (int c = 0; c < 4; c++) { /* 32 dims */
                            uint32_t w[4], f[4][2];
                            ldmatrix4(w, at + c * 512);
#pragma unroll
                            for (int x = 0; x < 4; x++) widen_e4m3x4(w[x], f[x][0], f[x][1]);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                mma16<true>(o[nt][2 * c], f[0][0], f[1][0], f[0][1], f[1][1], p[0][nt]);
                                mma16<true>(o[nt][2 * c + 1], f[2][0], f[3][0], f[2][1], f[3][1], p[0][nt]);
                            }
                        }
                    } else { /* transposed matrices: keys 0 .. 7 of dims 0 .. 7 and 8 .. 15, then keys 8 .. 15 */
                        const int j = 16 * k + r + 8 * (mi >> 1);
                        const uint32_t at = unit_u + 2 * BOX_BYTES + j * 128;
#pragma unroll
                        for (int d = 0; d < 8; d++) {
                            uint32_t w[4];
                            ldmatrix4_trans(w, at + (d >> 2) * BOX_BYTES + (((2 * (d & 3) + (mi & 1)) ^ (j & 7)) << 4));
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                mma16<false>(o[nt][d], w[0], w[1], w[2], w[3], p[0][nt]);
                                mma16<false>(o[nt][d], w[0], w[1], w[2], w[3], p[E4M3 ? 0 : 1][nt]);
                            }
                        }
                    }
                }
            }
            __syncwarp(); /* every lane has read the unit */
            if (i + WARPS < units) fetch(i + WARPS, next);
        }
        __syncthreads(); /* every warp has finished with its units: their states go there */
        float *mine = reinterpret_cast<float *>(smem) + warp * 8 * NT * PART;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int slot = 8 * nt + 2 * t + x;
                l[nt][x] = column_sum(l[nt][x]);
                if (g == 0) state_m[warp][slot] = m[nt][x], state_l[warp][slot] = l[nt][x];
                if (slot < slots)
#pragma unroll
                    for (int d = 0; d < 8; d++) mine[slot * PART + 16 * d + g] = o[nt][d][x], mine[slot * PART + 16 * d + 8 + g] = o[nt][d][2 + x];
            }
        __syncthreads();
        for (int slot = warp; slot < slots; slot += WARPS) { /* a warp per slot, four dimensions a lane */
            float top = state_m[0][slot], sum = 0.f;
#pragma unroll
            for (int w = 1; w < WARPS; w++) top = fmaxf(top, state_m[w][slot]);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float f = scale_of(state_m[w][slot], state_l[w][slot], top);
                const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(smem) + (w * 8 * NT + slot) * PART + 4 * lane);
                sum = fmaf(state_l[w][slot], f, sum);
                if (f != 0.f) x.x = fmaf(v.x, f, x.x), x.y = fmaf(v.y, f, x.y), x.z = fmaf(v.z, f, x.z), x.w = fmaf(v.w, f, x.w);
            }
            if (part_at < 0) {
                const float inv = sum > 0.f || sum != sum ? __fdiv_rn(1.f, E4M3 ? sum * P_SCALE : sum) : 0.f;
                *reinterpret_cast<uint2 *>((bf16 *)a.out + (first_row + slot / G) * a.ldo + (size_t)(kvh * G + slot % G) * HEAD_DIM + 4 * lane) =
                    make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
            } else {
                float *part = (float *)a.workspace + ((size_t)part_at * args.caps.small.slots + slot) * PART;
                if (lane == 0) part[0] = top, part[1] = sum;
                *reinterpret_cast<float4 *>(part + 4 + 4 * lane) = x;
            }
        }
        if (failed || whole) break; /* failed: the same for all, written before the barriers */
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); /* the states were written where the next units will be copied */
        __syncthreads();
    }
    if (args.caps.tiles) asm volatile("griddepcontrol.wait;" ::: "memory");
}

constexpr int MERGE_WARPS = 8, MERGE_SLOTS = 16;

/* Joins the states of N slots of an owner from `slot0` on: a warp, four dimensions a lane, TOGETHER states of each slot in flight. */
template <int N, int TOGETHER> __device__ __forceinline__ void join_slots(const ncb_paged &a, const Join &join, const float *parts, int part_slots, int slot0, int lane) {
    const int slots = min(N, join.slots - slot0), G = a.Hq / a.Hkv;
    if (slots <= 0) return;
    float top[N], sum[N];
    float4 y[N];
#pragma unroll
    for (int x = 0; x < N; x++) top[x] = -INFINITY, sum[x] = 0.f, y[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int b0 = join.first; b0 <= join.last; b0 += TOGETHER) {
        float2 ml[N][TOGETHER];
        float4 v[N][TOGETHER];
#pragma unroll
        for (int i = 0; i < TOGETHER; i++)
#pragma unroll
            for (int x = 0; x < N; x++) {
                ml[x][i] = make_float2(-INFINITY, 0.f), v[x][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (b0 + i > join.last || x >= slots) continue;
                const float *part = parts + ((size_t)(2 * (b0 + i) + (b0 + i == join.first)) * part_slots + slot0 + x) * PART;
                ml[x][i] = *reinterpret_cast<const float2 *>(part);
                v[x][i] = *reinterpret_cast<const float4 *>(part + 4 + 4 * lane);
            }
#pragma unroll
        for (int x = 0; x < N; x++) {
            float most = top[x];
#pragma unroll
            for (int i = 0; i < TOGETHER; i++) most = fmaxf(most, ml[x][i].x);
            const float old = scale_of(top[x], sum[x], most);
            top[x] = most, sum[x] *= old, y[x].x *= old, y[x].y *= old, y[x].z *= old, y[x].w *= old;
#pragma unroll
            for (int i = 0; i < TOGETHER; i++) {
                const float f = scale_of(ml[x][i].x, ml[x][i].y, most);
                sum[x] = fmaf(ml[x][i].y, f, sum[x]);
                if (f != 0.f) y[x].x = fmaf(v[x][i].x, f, y[x].x), y[x].y = fmaf(v[x][i].y, f, y[x].y), y[x].z = fmaf(v[x][i].z, f, y[x].z), y[x].w = fmaf(v[x][i].w, f, y[x].w);
            }
        }
    }
#pragma unroll
    for (int x = 0; x < N; x++) {
        if (x >= slots) break;
        const int slot = slot0 + x;
        const float inv = sum[x] > 0.f || sum[x] != sum[x] ? __fdiv_rn(1.f, a.e4m3 ? sum[x] * P_SCALE : sum[x]) : 0.f;
        *reinterpret_cast<uint2 *>((bf16 *)a.out + ((size_t)join.row + slot / G) * a.ldo + (size_t)(join.head * G + slot % G) * HEAD_DIM + 4 * lane) =
            make_uint2(pack_bf16(y[x].x * inv, y[x].y * inv), pack_bf16(y[x].z * inv, y[x].w * inv));
    }
}

/* The states of owners that were cut: a block per join of the schedule (and 16 of a tile's slots). Nothing but the record comes before the states, so that with few of them the
 * launch is as long as three reads one after the other: about 5 us behind the others, where finding an owner through the schedule's sums took 9 and with tiles' states 14. */
__global__ void __launch_bounds__(32 * MERGE_WARPS) k_paged_merge(const PagedArgs args) {
    const ncb_paged &a = args.p;
    const int smalls = args.caps.smalls && a.width > WHOLE_WIDTH ? args.caps.small.blocks : 0, tile = (int)blockIdx.x >= smalls, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const Class &cls = tile ? args.caps.tile : args.caps.small;
    const int groups = tile ? (cls.slots + MERGE_SLOTS - 1) / MERGE_SLOTS : 1, job = blockIdx.x - (tile ? smalls : 0);
    const float *parts = (const float *)a.workspace + parts_at(args.caps, tile);
    /* The next launch's blocks do not come before this one's have left: on SMs that still hold some of these they spread unevenly, and a call of 171 us that followed another
     * one took 240. */
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Join join = reinterpret_cast<const Join *>(a.work + class_at(args.caps, tile) + joins_at(cls))[job / groups];
    if (join.slots <= MERGE_WARPS) join_slots<1, 8>(a, join, parts, cls.slots, job % groups * MERGE_SLOTS + warp, lane);
    else join_slots<2, 4>(a, join, parts, cls.slots, job % groups * MERGE_SLOTS + 2 * warp, lane);
}

template <typename... Args> cudaError_t launch(void (*kernel)(Args...), unsigned grid, int threads, int smem, cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, Args(args)...);
}

/* Opts a kernel in to its dynamic shared memory, once per device, and asks for the split of an SM's memory that gives most to it: all kernels of a call do, so that an SM
 * on which the one before has not ended takes as many blocks as another. */
template <typename Kernel> cudaError_t allow_smem(Kernel kernel, int bytes, std::atomic<unsigned long long> &ready) {
    int device;
    cudaError_t rc = cudaGetDevice(&device);
    if (rc != cudaSuccess) return rc;
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (ready.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    rc = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (rc == cudaSuccess && bytes) rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (rc == cudaSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
    return rc;
}

template <bool E4M3, int NT, int WARPS> cudaError_t small(const CUtensorMap &map, const PagedArgs &args, long long blocks, cudaStream_t stream) {
    constexpr int smem = Unit<E4M3, WARPS>::SMEM;
    static std::atomic<unsigned long long> ready{0};
    const cudaError_t rc = allow_smem(k_paged_small<E4M3, NT, WARPS>, smem, ready);
    if (rc != cudaSuccess) return rc;
    return launch(k_paged_small<E4M3, NT, WARPS>, (unsigned)blocks, 32 * WARPS, smem, stream, map, args);
}
/* Where owners are whole and there is at most one for every SM, it has twelve warps in place of four: the call is then as long as its longest owner, not as
 * its bytes (three users of up to 700 positions, 10 heads, bf16: 8.7 us; four warps 13.5, four with three units under way each 12.0). */
template <bool E4M3, int NT> cudaError_t small(const CUtensorMap &map, const PagedArgs &args, cudaStream_t stream) {
    const bool whole = args.p.width <= WHOLE_WIDTH;
    const long long blocks = whole ? args.caps.small.owners * args.p.Hkv : args.caps.small.blocks;
    return whole && blocks <= args.p.blocks ? small<E4M3, NT, MANY>(map, args, blocks, stream) : small<E4M3, NT, FEW>(map, args, blocks, stream);
}
template <bool E4M3, bool TWICE> cudaError_t tile(const CUtensorMap &map_q, const CUtensorMap &map_kv, const PagedArgs &args, cudaStream_t stream) {
    constexpr int smem = tiles::Shape<E4M3>::SMEM;
    static std::atomic<unsigned long long> ready{0};
    const cudaError_t rc = allow_smem(tiles::k_paged_tiles<E4M3, TWICE>, smem, ready);
    if (rc != cudaSuccess) return rc;
    const long long whole = args.caps.tile.owners * args.p.Hkv; /* blocks where no tile is cut */
    return launch(tiles::k_paged_tiles<E4M3, TWICE>, (unsigned)(whole > args.caps.tile.blocks ? whole : args.caps.tile.blocks), tiles::THREADS, smem, stream, map_q, map_kv, args);
}

template <bool E4M3> cudaError_t tile(const CUtensorMap &map_q, const CUtensorMap &map_kv, const PagedArgs &args, cudaStream_t stream) {
    return args.p.max_fresh <= args.caps.tile.rows_per / 2 ? tile<E4M3, true>(map_q, map_kv, args, stream) : tile<E4M3, false>(map_q, map_kv, args, stream);
}

/* The queries as [rows][heads][128] in boxes of 64 columns, the heads of a group and the rows of a tile. */
bool query_map(const ncb_paged &a, int rows_per, CUtensorMap *out) {
    EncodeTiled encode = encoder();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)HEAD_DIM, (cuuint64_t)a.Hq, (cuuint64_t)a.rows}, strides[2] = {HEAD_DIM * 2, (cuuint64_t)a.ldq * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)(a.Hq / a.Hkv), (cuuint32_t)rows_per}, elem[3] = {1, 1, 1};
    return encode(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(a.q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

} /* namespace */

extern "C" {

int paged_attn_blocks(void) { return 148; } /* SMs */

long long paged_attn_workspace_bytes(int requests, long long rows, int width, int max_fresh, int Hq, int Hkv, int blocks) {
    if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || width <= 0 || !sizes_ok(requests, rows, max_fresh, Hq / Hkv, Hkv, blocks)) return -1;
    const Caps caps = caps_of(requests, rows, max_fresh, Hq / Hkv, blocks);
    return caps.tiles || width > WHOLE_WIDTH ? 4 * workspace_floats(caps) : 0;
}

int paged_attn(const ncb_paged *args, void *stream) {
    if (!args) return NCB_ERR_ARG;
    const ncb_paged &a = *args;
    if (a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv || a.width <= 0 || a.n_pages <= 0 || a.window < 0 || !(a.scale > 0.f)) return NCB_ERR_ARG;
    if (!sizes_ok(a.requests, a.rows, a.max_fresh, a.Hq / a.Hkv, a.Hkv, a.blocks)) return NCB_ERR_ARG;
    if (a.ldq < (long long)a.Hq * HEAD_DIM || a.ldo < (long long)a.Hq * HEAD_DIM) return NCB_ERR_ARG;
    if (a.rows == 0) return NCB_OK;
    if (!a.q || !a.pool || !a.out || !a.table || !a.work) return NCB_ERR_ARG;
    if (((uintptr_t)a.q | (uintptr_t)a.pool | (uintptr_t)a.out | (uintptr_t)a.workspace | (uintptr_t)a.work) % 16 || a.ldq % 8 || a.ldo % 8) return NCB_ERR_ALIGN;
    PagedArgs p = {a, caps_of(a.requests, a.rows, a.max_fresh, a.Hq / a.Hkv, a.blocks), a.scale * LOG2_E};
    const long long needed = paged_attn_workspace_bytes(a.requests, a.rows, a.width, a.max_fresh, a.Hq, a.Hkv, a.blocks);
    if (needed > 0 && !a.workspace) return NCB_ERR_ARG;
    if (a.workspace_bytes < needed) return NCB_ERR_WORKSPACE;
    const long long key_rows = (long long)a.n_pages * a.Hkv * 2 * PAGE_TOKENS;
    if (key_rows > 0x7fffffffll || p.caps.tile.owners * a.Hkv > 0x7fffffffll || p.caps.small.owners * a.Hkv > 0x7fffffffll) return NCB_ERR_UNSUPPORTED;
    CUtensorMap map = {}, map_q = {};
    const cudaStream_t s = (cudaStream_t)stream;
    if (p.caps.tiles) {
        if (!query_map(a, p.caps.tile.rows_per / 2, &map_q)) return NCB_ERR_LAUNCH;
        if (!a.e4m3 && !tensor_map(a.pool, (int)key_rows, HEAD_DIM, PAGE_TOKENS, &map)) return NCB_ERR_LAUNCH;
        if ((a.e4m3 ? tile<true>(map_q, map, p, s) : tile<false>(map_q, map, p, s)) != cudaSuccess) return NCB_ERR_LAUNCH;
    }
    if (p.caps.smalls) {
        if (!a.e4m3 && !tensor_map(a.pool, (int)key_rows, HEAD_DIM, BOX_ROWS, &map)) return NCB_ERR_LAUNCH;
        const bool one = p.caps.small.slots <= 8;
        const cudaError_t rc = a.e4m3 ? (one ? small<true, 1>(map, p, s) : small<true, 2>(map, p, s)) : (one ? small<false, 1>(map, p, s) : small<false, 2>(map, p, s));
        if (rc != cudaSuccess) return NCB_ERR_LAUNCH;
    }
    const int ends = (p.caps.smalls && a.width > WHOLE_WIDTH ? p.caps.small.blocks : 0) + (p.caps.tiles ? p.caps.tile.blocks * ((p.caps.tile.slots + MERGE_SLOTS - 1) / MERGE_SLOTS) : 0);
    if (ends == 0) return NCB_OK;
    static std::atomic<unsigned long long> ready{0};
    if (allow_smem(k_paged_merge, 0, ready) != cudaSuccess) return NCB_ERR_LAUNCH;
    return launch(k_paged_merge, ends, 32 * MERGE_WARPS, 0, s, p) == cudaSuccess ? NCB_OK : NCB_ERR_LAUNCH;
}

} /* extern "C" */
