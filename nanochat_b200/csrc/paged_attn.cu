/*
 * Attention of every request's new rows over its pages (page_plan.cu makes block tables and schedules, paged_append.cu fills the pages).
 * Replaces the reference's k_attn (model/kernels/decode.cu:567-675), which reads one slot's contiguous rows, for pools of pages,
 * grouped query heads, split lengths and several new rows per request.
 *
 * k_paged_split: a block takes one entry of the schedule and one key/value head: up to 64 query slots (new rows x the heads of the group) against a
 * run of the request's pages, which a fifth warp streams through a ring (TMA boxes of a bf16 page, one bulk copy of an e4m3 page).
 * Both contractions are m16n8k16 tensor-core MMAs with the query slots as M, in units of 16 keys: the score accumulators are already
 * the A operand of P V. Of at most 16 slots every warp has a quarter of each page's keys, of at most 32 a pair of warps has half of
 * them each, else every warp has 16 slots and all keys; each keeps its own maximum, sum and output, joined through shared memory at the end.
 *   - bf16 pages: probabilities enter P V as two bf16 terms (hi + lo, 16 bits): one term would double the error of the bf16 output,
 *     and the stream of pages leaves the MMAs time;
 *   - e4m3 pages: bytes widened to f16 (exact) in registers, queries f16 after a power-of-two scale (exact down to 2^-24 of a row's
 *     largest), the key's scale on the fp32 score, the value's folded into the f16 probability (11 bits), the running maximum that of score +
 *     log2(value scale), as in decode_attn.cu. Key columns are permuted so that a lane's probabilities are those of four consecutive bytes of V^T.
 * What a row does not see must not reach it, not even as zero times a NaN or an infinity: scores are masked by selects, and a unit that is not
 * seen whole by every slot has its values looked at; if one is not finite, its products are made row by row over the keys seen.
 *
 * k_paged_merge: the states of owners that were cut, one warp per query slot.
 * Waits are bounded: when one expires NCB_DEV_WAIT_TIMEOUT is flagged and the block leaves after its copies in flight.
 */
#include "paged_tiles.cuh"

namespace {

using namespace paged;

constexpr int SPLIT_WARPS = 4, SPLIT_THREADS = 32 * (SPLIT_WARPS + 1);
constexpr int BLOCKS_PER_SM = 2;
constexpr float LOG2_E = 1.4426950408889634f;
constexpr float P_SCALE = 256.f; /* keeps small folded probabilities among f16's normal numbers; an exact power of two */
constexpr float MIN_LOG2_VSCALE = -64.f;
constexpr int WIDE_PAGE_BYTES = 2 * PAGE_TOKENS * HEAD_DIM * 2, BOX_BYTES = 2 * PAGE_TOKENS * 128; /* a bf16 page: two boxes of 64 columns, keys above values */

template <bool E4M3> struct Ring {
    static constexpr int STAGE = E4M3 ? PAGE_BYTES : WIDE_PAGE_BYTES, STAGES = E4M3 ? 6 : 3;
    static constexpr int SMEM = 1024 + STAGE * STAGES; /* 1024: swizzled boxes are aligned by hand */
    static_assert(BLOCKS_PER_SM * (SMEM + 2048) <= 228 * 1024, "blocks per SM");
    static_assert(SPLIT_WARPS * 16 * PART * 4 <= STAGE * STAGES, "the warps' states reuse the ring");
};

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool F16> __device__ __forceinline__ void mma16(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t *r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t *r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bulk_load_once(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy) : "memory");
}

/* What a state (m, l) counts relative to 2^top: nothing where it holds nothing. */
__device__ __forceinline__ float scale_of(float m, float l, float top) { return m == -INFINITY && l == l ? 0.f : ex2(m - top); }

/* Value `dim` of in-page position j. */
template <bool E4M3> __device__ __forceinline__ float value_at(const uint8_t *page, int j, int dim) {
    if (E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw(page[page_v_byte(j, dim)], __NV_E4M3)));
    const int r = PAGE_TOKENS + j;
    return __bfloat162float(*reinterpret_cast<const bf16 *>(page + dim / 64 * BOX_BYTES + r * 128 + ((dim % 64 / 8 ^ r & 7) * 16) + dim % 8 * 2));
}

/* Whether some value of the 16 positions from `key` is infinite or NaN (a warp). */
template <bool E4M3> __device__ __forceinline__ bool strange_values(const uint8_t *page, int key, int lane) {
    bool strange = false;
    if (E4M3) { /* 2,048 bytes, a position's codes at the same byte of 128 chunks; NaN is 0x7f with either sign */
        const uint4 *v = reinterpret_cast<const uint4 *>(page + page_v_byte(key, 0));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 x = v[lane + 32 * i];
#pragma unroll
            for (int e = 0; e < 4; e++) strange |= __vcmpeq4((&x.x)[e] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
        }
    } else {
        const int r = PAGE_TOKENS + key + (lane >> 1); /* half a row a lane: one box */
        const uint4 *v = reinterpret_cast<const uint4 *>(page + (lane & 1) * BOX_BYTES + r * 128);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t acc = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"((&v[i].x)[e]), "r"(0u));
            strange |= (acc & 0x7fff7fffu) != 0;
        }
    }
    return __any_sync(0xffffffffu, strange);
}

template <bool E4M3> __global__ void __launch_bounds__(SPLIT_THREADS, BLOCKS_PER_SM) k_paged_split(const __grid_constant__ CUtensorMap map, const PagedArgs args) {
    using R = Ring<E4M3>;
    extern __shared__ __align__(128) uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[2 * R::STAGES];
    __shared__ int in_pool[R::STAGES]; /* the stage holds a page */
    __shared__ int failed;
    __shared__ float state_m[SPLIT_WARPS][16], state_l[SPLIT_WARPS][16];
    const ncb_paged &a = args.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t *smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const uint32_t ring = smem_u32(smem);
    auto full = [&](int st) { return smem_u32(bars + st); };
    auto empty = [&](int st) { return smem_u32(bars + R::STAGES + st); };
    if (tid == 0) {
        for (int st = 0; st < R::STAGES; st++) {
            mbar_init(full(st), 1);
            mbar_init(empty(st), SPLIT_WARPS);
        }
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int G = a.Hq / a.Hkv, jobs = a.work[0] * a.Hkv;
    int base = 0; /* pages that have been through the ring */
    for (int job = blockIdx.x; job < jobs; job += gridDim.x) {
    const int kvh = job % a.Hkv;
    const Entry e = reinterpret_cast<const Entry *>(a.work + entries_at(args.caps, 0))[job / a.Hkv];
    const int served = a.served[e.request], slots = e.rows * G, n = e.page1 - e.page0;
    const int first_pos = a.lens[e.request] - served + e.row0, last_pos = first_pos + e.rows - 1;
    const long long first_row = a.row_start[e.request] + e.row0;
    auto begin_of = [&](int pos) { return a.window > 0 ? max(0, pos + 1 - a.window) : 0; }; /* the first position that the row at pos sees */

    if (warp == SPLIT_WARPS) {
        if (lane == 0) { /* copies */
            const int *table = a.table + (size_t)e.request * a.width + e.page0;
            uint64_t once = policy_evict_first();
            int sent = 0, page = n > 0 ? table[0] : 0;
            for (int i = 0; i < n; i++) {
                const int at = base + i, st = at % R::STAGES, next = i + 1 < n ? table[i + 1] : 0;
                if (at >= R::STAGES && !mbar_wait(empty(st), (at / R::STAGES - 1) & 1)) {
                    flag(a.status, NCB_DEV_WAIT_TIMEOUT);
                    failed = 1;
                    break;
                }
                const bool ok = (unsigned)page < (unsigned)a.n_pages;
                in_pool[st] = ok;
                if (!ok) {
                    flag(a.status, NCB_DEV_BAD_PAGE);
                    arrive(full(st));
                } else if (E4M3) {
                    mbar_expect_tx(full(st), PAGE_BYTES);
                    bulk_load_once(ring + st * R::STAGE, (const uint8_t *)a.pool + ((size_t)page * a.Hkv + kvh) * PAGE_BYTES, PAGE_BYTES, full(st), once);
                } else {
                    mbar_expect_tx(full(st), WIDE_PAGE_BYTES);
                    const int row = (page * a.Hkv + kvh) * 2 * PAGE_TOKENS;
                    tma_load(ring + st * R::STAGE, &map, 0, row, full(st), once);
                    tma_load(ring + st * R::STAGE + BOX_BYTES, &map, 64, row, full(st), once);
                }
                sent++;
                page = next;
            }
            if (failed) /* nobody leaves under a copy */
                for (int at = base + max(0, sent - R::STAGES); at < base + sent; at++) mbar_wait(full(at % R::STAGES), (at / R::STAGES) & 1);
        }
        __syncwarp();
    } else {
        /* this warp's 16 slots from 16 group, and its units of 16 keys of every page */
        const int groups = (slots + 15) / 16, share = groups == 1 ? 4 : groups == 2 ? 2 : 1; /* warps that share a group */
        const int group = warp / share, unit0 = warp % share * (4 / share), unit1 = unit0 + 4 / share;
        const bool has_slots = group < groups;
        const int g = lane >> 2, t = lane & 3;
        uint32_t qa[8][4];
        float factor[2];
        int seen_from[2], seen_to[2]; /* positions that slots g and g + 8 see: [from, to] */
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int slot = 16 * group + g + 8 * r;
            const bool on = slot < slots;
            const int i = on ? slot / G : e.rows - 1; /* slots without a row see what the last one does */
            const bf16 *src = (const bf16 *)a.q + (first_row + i) * a.ldq + (size_t)(kvh * G + (on ? slot % G : 0)) * HEAD_DIM;
            seen_to[r] = first_pos + i, seen_from[r] = begin_of(seen_to[r]);
            factor[r] = args.scale_log2;
            if (E4M3) { /* k slots (2t, 2t+1) and (2t+8, 2t+9) of step s are dims 16 s + 4 t .. + 3, as the cache bytes arrive */
                float amax = 0.f;
                uint2 u[8];
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    u[s] = on ? *reinterpret_cast<const uint2 *>(src + 16 * s + 4 * t) : make_uint2(0u, 0u);
                    amax = fmaxf(amax, fmaxf(fmaxf(fabsf(__uint_as_float(u[s].x << 16)), fabsf(__uint_as_float(u[s].x & 0xffff0000u))),
                                             fmaxf(fabsf(__uint_as_float(u[s].y << 16)), fabsf(__uint_as_float(u[s].y & 0xffff0000u)))));
                }
                amax = quad_max(amax);
                /* the row's largest magnitude to [2^14, 2^15): what f16 then rounds or loses is below 2^-38 of it */
                const int expo = (int)((__float_as_uint(amax) >> 23) & 0xffu) - 127, down = max(-100, min(expo - 14, 112));
                const float mul = __uint_as_float((uint32_t)(127 - down) << 23), back = __uint_as_float((uint32_t)(127 + down) << 23);
                factor[r] *= back;
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    qa[s][r] = pack_f16(__uint_as_float(u[s].x << 16) * mul, __uint_as_float(u[s].x & 0xffff0000u) * mul);
                    qa[s][2 + r] = pack_f16(__uint_as_float(u[s].y << 16) * mul, __uint_as_float(u[s].y & 0xffff0000u) * mul);
                }
            } else {
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    qa[s][r] = on ? *reinterpret_cast<const uint32_t *>(src + 16 * s + 2 * t) : 0u;
                    qa[s][2 + r] = on ? *reinterpret_cast<const uint32_t *>(src + 16 * s + 8 + 2 * t) : 0u;
                }
            }
        }
        const int all_from = begin_of(last_pos), all_to = first_pos; /* what every slot of the block sees */
        const int any_from = begin_of(first_pos);
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[16][4];
#pragma unroll
        for (int d = 0; d < 16; d++)
#pragma unroll
            for (int x = 0; x < 4; x++) o[d][x] = 0.f;

        for (int i = 0; i < n; i++) {
            const int at = base + i, st = at % R::STAGES;
            if (!__all_sync(0xffffffffu, mbar_wait(full(st), (at / R::STAGES) & 1))) {
                if (lane == 0) flag(a.status, NCB_DEV_WAIT_TIMEOUT), failed = 1;
                break;
            }
            const uint8_t *page = smem + st * R::STAGE;
            const uint32_t page_u = ring + st * R::STAGE;
            const int page_pos = (e.page0 + i) * PAGE_TOKENS;
            const bool here = has_slots && in_pool[st];
            for (int unit = unit0; here && unit < unit1; unit++) {
                const int key0 = 16 * unit, pos0 = page_pos + key0;
                if (pos0 > last_pos || pos0 + 15 < any_from) continue;
                const bool masked = pos0 < all_from || pos0 + 15 > all_to;
                /* ---- scores: of key tile c, element x: slot g + 8 (x / 2), key key0 + 8 c + 2 t + x % 2, or (E4M3) 4 t + 2 c + x % 2 ---- */
                float s[2][4] = {};
                if (E4M3) {
                    const int mi = lane >> 3, r = lane & 7, j = key0 + 4 * (r >> 1) + 2 * (mi & 1) + (r & 1);
                    const uint32_t row = page_u + PAGE_K + j * HEAD_DIM, swz = (uint32_t)((j >> 2) & 7);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t kr[4], b[2];
                        ldmatrix4(kr, row + (((2 * k + (mi >> 1)) ^ swz) << 4));
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            widen_e4m3x4(kr[x], b[0], b[1]);
                            mma16<true>(s[x & 1], qa[2 * k + (x >> 1)], b[0], b[1]);
                        }
                    }
                } else {
                    const int mi = lane >> 3, j = key0 + (mi >> 1) * 8 + (lane & 7);
                    const uint32_t row = page_u + j * 128;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        uint32_t kr[4];
                        ldmatrix4(kr, row + (k >> 2) * BOX_BYTES + (((2 * (k & 3) + (mi & 1)) ^ (j & 7)) << 4));
                        mma16<false>(s[0], qa[k], kr[0], kr[1]);
                        mma16<false>(s[1], qa[k], kr[2], kr[3]);
                    }
                }
                float vscale[2][2] = {{1.f, 1.f}, {1.f, 1.f}}, lv[2][2] = {{0.f, 0.f}, {0.f, 0.f}}; /* of this lane's keys [c][x % 2] */
                if (E4M3) {
                    const float4 k4 = *reinterpret_cast<const float4 *>(page + PAGE_KS + (key0 + 4 * t) * 4);
                    const float4 v4 = *reinterpret_cast<const float4 *>(page + PAGE_VS + (key0 + 4 * t) * 4);
                    const float ks[2][2] = {{k4.x, k4.y}, {k4.z, k4.w}};
                    vscale[0][0] = v4.x, vscale[0][1] = v4.y, vscale[1][0] = v4.z, vscale[1][1] = v4.w;
#pragma unroll
                    for (int c = 0; c < 2; c++)
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            s[c][x] *= ks[c][x], s[c][2 + x] *= ks[c][x];
                            lv[c][x] = fmaxf(lg2(vscale[c][x]), MIN_LOG2_VSCALE);
                        }
                }
                auto seen = [&](int c, int x) {
                    const int pos = pos0 + (E4M3 ? 4 * t + 2 * c : 8 * c + 2 * t) + (x & 1);
                    return !masked || (pos >= seen_from[x >> 1] && pos <= seen_to[x >> 1]);
                };
                float top[2];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    float best = -INFINITY;
#pragma unroll
                    for (int c = 0; c < 2; c++)
#pragma unroll
                        for (int x = 2 * r; x < 2 * r + 2; x++) {
                            s[c][x] *= factor[r];
                            best = fmaxf(best, seen(c, x) ? s[c][x] + lv[c][x & 1] : -INFINITY);
                        }
                    top[r] = fmaxf(quad_max(best), m[r]);
                }
                if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) { /* some slot's maximum moved: rescale */
                    const float c0 = m[0] == -INFINITY ? 0.f : ex2(m[0] - top[0]), c1 = m[1] == -INFINITY ? 0.f : ex2(m[1] - top[1]);
                    l[0] *= c0, l[1] *= c1;
#pragma unroll
                    for (int d = 0; d < 16; d++) o[d][0] *= c0, o[d][1] *= c0, o[d][2] *= c1, o[d][3] *= c1;
                    m[0] = top[0], m[1] = top[1];
                }
                float p[2][4];
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const bool counts = seen(c, x) && (top[x >> 1] != -INFINITY || s[c][x] != s[c][x]); /* a row of NaN scores stays NaN */
                        const float w = counts ? ex2(s[c][x] - top[x >> 1]) : 0.f;
                        l[x >> 1] += w;
                        p[c][x] = !E4M3 ? w : counts ? w * (vscale[c][x & 1] * P_SCALE) : 0.f;
                    }
                if (masked && strange_values<E4M3>(page, key0, lane)) { /* rare: row by row, over the keys that the row sees */
#pragma unroll 1
                    for (int j = 0; j < 16; j++) {
                        const int c = E4M3 ? (j & 3) >> 1 : j >> 3, from = E4M3 ? j >> 2 : (j & 7) >> 1, pos = pos0 + j;
                        float w[2];
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            const float even = c ? p[1][2 * r] : p[0][2 * r], odd = c ? p[1][2 * r + 1] : p[0][2 * r + 1];
                            w[r] = __shfl_sync(0xffffffffu, (j & 1) ? odd : even, (lane & ~3) | from);
                        }
#pragma unroll
                        for (int r = 0; r < 2; r++)
                            if (pos >= seen_from[r] && pos <= seen_to[r])
#pragma unroll
                                for (int d = 0; d < 16; d++) {
                                    o[d][2 * r] = fmaf(w[r], value_at<E4M3>(page, key0 + j, 8 * d + 2 * t), o[d][2 * r]);
                                    o[d][2 * r + 1] = fmaf(w[r], value_at<E4M3>(page, key0 + j, 8 * d + 2 * t + 1), o[d][2 * r + 1]);
                                }
                    }
                    continue;
                }
                /* ---- values ---- */
                if (E4M3) {
                    const uint32_t pa[4] = {pack_f16(p[0][0], p[0][1]), pack_f16(p[0][2], p[0][3]), pack_f16(p[1][0], p[1][1]), pack_f16(p[1][2], p[1][3])};
                    const uint32_t at = page_u + page_v_byte(key0, 0) + lane * 16;
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        uint32_t vr[4], b[2];
                        ldmatrix4(vr, at + d * 512);
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            widen_e4m3x4(vr[x], b[0], b[1]);
                            mma16<true>(o[4 * d + x], pa, b[0], b[1]);
                        }
                    }
                } else {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int c = 0; c < 2; c++)
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            const float x = p[c][2 * r], y = p[c][2 * r + 1];
                            hi[2 * c + r] = pack_bf16(x, y);
                            lo[2 * c + r] = pack_bf16(x - __uint_as_float(hi[2 * c + r] << 16), y - __uint_as_float(hi[2 * c + r] & 0xffff0000u));
                        }
                    const int mi = lane >> 3, j = PAGE_TOKENS + key0 + (mi & 1) * 8 + (lane & 7);
                    const uint32_t row = page_u + j * 128;
#pragma unroll
                    for (int d = 0; d < 8; d++) { /* 16 value columns at a time */
                        uint32_t vr[4];
                        ldmatrix4_trans(vr, row + (d >> 2) * BOX_BYTES + (((2 * (d & 3) + (mi >> 1)) ^ (j & 7)) << 4));
                        mma16<false>(o[2 * d], hi, vr[0], vr[1]);
                        mma16<false>(o[2 * d + 1], hi, vr[2], vr[3]);
                        mma16<false>(o[2 * d], lo, vr[0], vr[1]);
                        mma16<false>(o[2 * d + 1], lo, vr[2], vr[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) arrive(empty(st));
        }
        l[0] = quad_sum(l[0]), l[1] = quad_sum(l[1]);
        /* every warp of the block has finished with the ring before its states are written there */
        asm volatile("bar.sync 1, 128;" ::: "memory");
        float *mine = reinterpret_cast<float *>(smem) + warp * 16 * PART;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            if (t == 0) state_m[warp][g + 8 * r] = m[r], state_l[warp][g + 8 * r] = has_slots ? l[r] : 0.f;
#pragma unroll
            for (int d = 0; d < 16; d++) *reinterpret_cast<float2 *>(mine + (g + 8 * r) * PART + 8 * d + 2 * t) = make_float2(o[d][2 * r], o[d][2 * r + 1]);
        }
    }
    __syncthreads();
    if (tid < HEAD_DIM) { /* a thread per dimension */
        const int groups = (slots + 15) / 16, share = groups == 1 ? 4 : groups == 2 ? 2 : 1;
        for (int slot = 0; slot < slots; slot++) {
            const int w0 = slot / 16 * share, r = slot % 16;
            float top = -INFINITY, sum = 0.f, x = 0.f;
            for (int w = w0; w < w0 + share; w++) top = fmaxf(top, state_m[w][r]);
            for (int w = w0; w < w0 + share; w++) {
                const float f = scale_of(state_m[w][r], state_l[w][r], top);
                sum = fmaf(state_l[w][r], f, sum);
                if (f != 0.f) x = fmaf(reinterpret_cast<const float *>(smem)[(w * 16 + r) * PART + tid], f, x);
            }
            const long long row = first_row + slot / G;
            const int head = kvh * G + slot % G;
            if (e.part < 0) {
                const float inv = sum > 0.f || sum != sum ? __fdiv_rn(1.f, E4M3 ? sum * P_SCALE : sum) : 0.f;
                ((bf16 *)a.out)[row * a.ldo + (size_t)head * HEAD_DIM + tid] = __float2bfloat16_rn(x * inv);
            } else {
                float *part = (float *)a.workspace + ((size_t)((long long)e.part * a.Hkv + kvh) * args.caps.split.slots + slot) * PART;
                if (tid == 0) part[0] = top, part[1] = sum;
                part[4 + tid] = x;
            }
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); /* the states were written where the next pages will be copied */
    __syncthreads();
    if (failed) break;
    base += n;
    }
}

constexpr int MERGE_WARPS = 4;

/* A warp per query slot of an owner that was cut; lanes have four dimensions each. */
__global__ void __launch_bounds__(32 * MERGE_WARPS) k_paged_merge(const PagedArgs args) {
    const ncb_paged &a = args.p;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, G = a.Hq / a.Hkv, warps = gridDim.x * MERGE_WARPS;
    long long job = (long long)blockIdx.x * MERGE_WARPS + threadIdx.x / 32;
    for (int tile = 0; tile <= args.caps.tiles; tile++) {
        const Class &cls = tile ? args.caps.tile : args.caps.split;
        const Merge *merges = reinterpret_cast<const Merge *>(a.work + merges_at(args.caps, tile));
        const float *parts = (const float *)a.workspace + parts_at(args.caps, a.Hkv, tile);
        const long long jobs = (long long)a.work[2 * tile + 1] * a.Hkv * cls.slots;
        for (; job < jobs; job += warps) {
            const int slot = (int)(job % cls.slots), kvh = (int)(job / cls.slots % a.Hkv);
            const Merge e = merges[job / cls.slots / a.Hkv];
            if (slot >= e.rows * G) continue;
            const float *part = parts + ((size_t)((long long)e.part * a.Hkv + kvh) * cls.slots + slot) * PART;
            const size_t step = (size_t)a.Hkv * cls.slots * PART;
            float top = -INFINITY, sum = 0.f;
            for (int c = lane; c < e.parts; c += 32) top = fmaxf(top, part[c * step]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int c = 0; c < e.parts; c++) {
                const float2 ml = *reinterpret_cast<const float2 *>(part + c * step);
                const float4 v = *reinterpret_cast<const float4 *>(part + c * step + 4 + 4 * lane);
                const float f = scale_of(ml.x, ml.y, top);
                sum = fmaf(ml.y, f, sum);
                if (f != 0.f) x.x = fmaf(v.x, f, x.x), x.y = fmaf(v.y, f, x.y), x.z = fmaf(v.z, f, x.z), x.w = fmaf(v.w, f, x.w);
            }
            const float inv = sum > 0.f || sum != sum ? __fdiv_rn(1.f, a.e4m3 ? sum * P_SCALE : sum) : 0.f;
            const uint2 y = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
            *reinterpret_cast<uint2 *>((bf16 *)a.out + (e.row + slot / G) * a.ldo + (size_t)(kvh * G + slot % G) * HEAD_DIM + 4 * lane) = y;
        }
        job -= jobs;
    }
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

template <bool E4M3> cudaError_t split(const CUtensorMap &map, const PagedArgs &args, cudaStream_t stream) {
    constexpr int smem = Ring<E4M3>::SMEM;
    const cudaError_t rc = cudaFuncSetAttribute(k_paged_split<E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc != cudaSuccess) return rc;
    const long long jobs = args.caps.split.entries * args.p.Hkv;
    return launch(k_paged_split<E4M3>, (unsigned)(jobs < args.p.blocks ? jobs : args.p.blocks), SPLIT_THREADS, smem, stream, map, args);
}
template <bool E4M3> cudaError_t tile(const CUtensorMap &map_q, const CUtensorMap &map_kv, const PagedArgs &args, cudaStream_t stream) {
    constexpr int smem = tiles::Shape<E4M3>::SMEM;
    const cudaError_t rc = cudaFuncSetAttribute(tiles::k_paged_tiles<E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc != cudaSuccess) return rc;
    return launch(tiles::k_paged_tiles<E4M3>, (unsigned)(args.caps.tile.entries * args.p.Hkv), E4M3 ? tiles::THREADS : 32 * tiles::WIDEN_WARP, smem, stream, map_q, map_kv, args);
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

int paged_attn_blocks(void) { return BLOCKS_PER_SM * 148; }

long long paged_attn_workspace_bytes(int requests, long long rows, int max_fresh, int Hq, int Hkv, int blocks) {
    if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || !sizes_ok(requests, rows, max_fresh, Hq / Hkv, Hkv, blocks)) return -1;
    const Caps c = caps_of(requests, rows, max_fresh, Hq / Hkv, Hkv, blocks);
    return 4 * workspace_floats(c, Hkv);
}

int paged_attn(const ncb_paged *args, void *stream) {
    if (!args) return NCB_ERR_ARG;
    const ncb_paged &a = *args;
    if (a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv || a.width <= 0 || a.n_pages <= 0 || a.window < 0 || !(a.scale > 0.f)) return NCB_ERR_ARG;
    if (!sizes_ok(a.requests, a.rows, a.max_fresh, a.Hq / a.Hkv, a.Hkv, a.blocks)) return NCB_ERR_ARG;
    if (a.ldq < (long long)a.Hq * HEAD_DIM || a.ldo < (long long)a.Hq * HEAD_DIM) return NCB_ERR_ARG;
    if (a.rows == 0) return NCB_OK;
    if (!a.q || !a.pool || !a.out || !a.workspace || !a.table || !a.row_start || !a.served || !a.lens || !a.work) return NCB_ERR_ARG;
    if (((uintptr_t)a.q | (uintptr_t)a.pool | (uintptr_t)a.out | (uintptr_t)a.workspace | (uintptr_t)a.work) % 16 || a.ldq % 8 || a.ldo % 8) return NCB_ERR_ALIGN;
    PagedArgs p = {a, caps_of(a.requests, a.rows, a.max_fresh, a.Hq / a.Hkv, a.Hkv, a.blocks), a.scale * LOG2_E};
    if (a.workspace_bytes < paged_attn_workspace_bytes(a.requests, a.rows, a.max_fresh, a.Hq, a.Hkv, a.blocks)) return NCB_ERR_WORKSPACE;
    const long long key_rows = (long long)a.n_pages * a.Hkv * 2 * PAGE_TOKENS;
    if (key_rows > 0x7fffffffll || p.caps.split.entries * a.Hkv > 0x7fffffffll || p.caps.tile.entries * a.Hkv > 0x7fffffffll) return NCB_ERR_UNSUPPORTED;
    CUtensorMap map = {}, map_q = {}, map_tile = {};
    if (!a.e4m3 && !tensor_map(a.pool, (int)key_rows, HEAD_DIM, 2 * PAGE_TOKENS, &map)) return NCB_ERR_LAUNCH;
    const cudaStream_t s = (cudaStream_t)stream;
    if (p.caps.tiles) {
        if (!query_map(a, p.caps.tile.rows_per, &map_q)) return NCB_ERR_LAUNCH;
        if (!a.e4m3 && !tensor_map(a.pool, (int)key_rows, HEAD_DIM, PAGE_TOKENS, &map_tile)) return NCB_ERR_LAUNCH;
        if ((a.e4m3 ? tile<true>(map_q, map_tile, p, s) : tile<false>(map_q, map_tile, p, s)) != cudaSuccess) return NCB_ERR_LAUNCH;
    }
    if ((a.e4m3 ? split<true>(map, p, s) : split<false>(map, p, s)) != cudaSuccess) return NCB_ERR_LAUNCH;
    return launch(k_paged_merge, 4 * 148, 32 * MERGE_WARPS, 0, s, p) == cudaSuccess ? NCB_OK : NCB_ERR_LAUNCH;
}

} /* extern "C" */
