/*
 * paged_append: kv_append.cu's operator for a pool of pages, where a row's k and v go to a place (page * 64 + position % 64) instead of a
 * position of a slot: the same row arithmetic (kv_row.cuh), so the same q bits, cache bytes and scales; for bf16 pools the rotated keys
 * and the values are stored as they are. Replaces the reference's k_prologue (model/kernels/decode.cu:551-565) for such pools.
 *
 * One head row of 128 values by 8 lanes; a 128-thread block holds the same head row of 16 consecutive rows of the step and
 * walks over several head rows. A run of 16 rows whose places share a 16-byte chunk of V (a multiple of 16 and the 15 after it) has
 * its e4m3 V bytes transposed through shared memory and stored as 128 chunks by the block in whose rows it begins; other rows store them
 * byte by byte. A page's places are consecutive exactly where a request's positions are, so the places alone decide.
 *
 * Bound by the latency of its loads and, in decode steps, of the launch: a warp has one head row's inputs under way while it works on another, so blocks per SM count
 * most (bf16 pages, 8,184 rows of 32 + 8 + 8 heads: 9, 8, 7, 6 blocks 41.1, 37.5, 38.0, 40.6 us; a second head row under way instead 38.8 at 7 blocks, 45.8 at the 5 that
 * need no spills). A row's cosines and sines stay in registers for all its heads: 39.8 -> 37.5 us (5.4 TB/s; e4m3 pages 46.9 -> 45.7), 2,046 rows 12.4 -> 10.7.
 * 64 rows of a decode step: 5.1 us (e4m3), 2.5 us (bf16).
 */
#include "kv_row.cuh"

namespace {

constexpr int BLOCK = 128, ROWS_PER_BLOCK = BLOCK / LANES;

struct AppendArgs {
    const bf16 *qkv;
    const float *q_gain, *k_gain, *cs, *sn;
    const int32_t *pos, *place;
    bf16 *q_out;
    uint8_t *pool;
    long long rows, stride;
    int Hq, Hkv, table_len, n_pages, heads_per_block;
    int *status;
};

template <bool E4M3> __global__ void __launch_bounds__(BLOCK, E4M3 ? 7 : 8) k_paged_append(const AppendArgs a) {
    constexpr int BACK = ROWS_PER_BLOCK - 1, NEAR = ROWS_PER_BLOCK + 2 * BACK; /* rows whose places decide about this block's */
    __shared__ __align__(16) uint8_t vt[E4M3 ? HEAD_DIM : 1][ROWS_PER_BLOCK];   /* a run's V transposed: [dim][position] */
    __shared__ int near_place[NEAR], start_of;
    __shared__ uint32_t links[2];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int g = threadIdx.x / LANES, t = threadIdx.x % LANES, o = t * VEC;
    const long long row0 = (long long)blockIdx.x * ROWS_PER_BLOCK, row = row0 + g;
    if (threadIdx.x < NEAR) { /* the place of a row that is stored, else -2 (which nothing follows) */
        const long long r = row0 - BACK + threadIdx.x;
        int place = -2;
        if (r >= 0 && r < a.rows) {
            const int p = a.pos[r];
            place = a.place[r];
            if (p < 0 || place < 0 || p >= a.table_len || place / PAGE_TOKENS >= a.n_pages) {
                if (p >= 0 && place >= 0 && r >= row0 && r < row0 + ROWS_PER_BLOCK && blockIdx.y == 0) flag(a.status, NCB_DEV_BAD_POSITION);
                place = -2;
            }
        }
        near_place[threadIdx.x] = place;
    }
    if (threadIdx.x == 0) start_of = -1;
    __syncthreads();
    if (threadIdx.x < 64) { /* bit i: row i + 1's place follows row i's */
        const int i = threadIdx.x;
        const uint32_t bits = __ballot_sync(0xffffffffu, i + 1 < NEAR && near_place[i] >= 0 && near_place[i + 1] == near_place[i] + 1);
        if ((i & 31) == 0) links[i >> 5] = bits;
    }
    __syncthreads();
    const unsigned long long link = (unsigned long long)links[1] << 32 | links[0];
    const int place = near_place[BACK + g];
    const bool on = place >= 0; /* the same for the 8 lanes of a row; nobody leaves before the last barrier */
    const bool grouped = E4M3 && on && (link >> (BACK + g - place % ROWS_PER_BLOCK) & 0x7fff) == 0x7fff;
    if (grouped && place % ROWS_PER_BLOCK == 0 && t == 0) start_of = g;
    __syncthreads();
    const int start = start_of, v_first = a.Hq + a.Hkv, first = blockIdx.y * a.heads_per_block, last = min(first + a.heads_per_block, a.Hq + 2 * a.Hkv);
    uint4 raw1 = make_uint4(0, 0, 0, 0), raw2 = raw1;
    auto load = [&](const bf16 *x, int which) {
        raw1 = *reinterpret_cast<const uint4 *>(x + (size_t)which * HEAD_DIM);
        raw2 = *reinterpret_cast<const uint4 *>(x + (size_t)which * HEAD_DIM + HALF);
    };
    auto page_of = [&](int at, int head) { return a.pool + ((size_t)(at / PAGE_TOKENS) * a.Hkv + head) * PAGE_BYTES; };
    auto wide_row = [&](int at, int head, int side) { /* a bf16 page: [2][64][128] */
        return reinterpret_cast<bf16 *>(a.pool) + (((size_t)(at / PAGE_TOKENS) * a.Hkv + head) * 2 + side) * PAGE_TOKENS * HEAD_DIM + at % PAGE_TOKENS * HEAD_DIM;
    };
    if (on && first < v_first) { /* q and k heads: every row by its own 8 lanes */
        const bf16 *x = a.qkv + row * a.stride + o;
        const size_t tab = (size_t)a.pos[row] * HALF;
        const int j = place % PAGE_TOKENS, end = min(last, v_first);
        const float4 *cos_at = reinterpret_cast<const float4 *>(a.cs + tab + o), *sin_at = reinterpret_cast<const float4 *>(a.sn + tab + o);
        const float4 cos[2] = {cos_at[0], cos_at[1]}, sin[2] = {sin_at[0], sin_at[1]}; /* of all its head rows; left in memory they are read again for each, since the stores between might change them */
        load(x, first);
        for (int which = first; which < end; which++) {
            float x1[VEC], x2[VEC];
            unpack_bf16x8(raw1, x1);
            unpack_bf16x8(raw2, x2);
            if (which + 1 < end) load(x, which + 1); /* the next head row's inputs start now */
            const bool is_q = which < a.Hq;
            norm_rotate_by(x1, x2, is_q ? a.q_gain : a.k_gain, o, [&](int q) { return cos[q / 4]; }, [&](int q) { return sin[q / 4]; });
            if (is_q || !E4M3) {
                bf16 *to = is_q ? a.q_out + ((size_t)row * a.Hq + which) * HEAD_DIM : wide_row(place, which - a.Hq, 0);
                *reinterpret_cast<uint4 *>(to + o) = pack_bf16x8(x1);
                *reinterpret_cast<uint4 *>(to + HALF + o) = pack_bf16x8(x2);
            } else {
                uint8_t b1[VEC], b2[VEC], *page = page_of(place, which - a.Hq);
                const float scale = quantise(x1, x2, b1, b2);
                if (t == 0) reinterpret_cast<float *>(page + PAGE_KS)[j] = scale;
                store_k_row16(page, j, t, b1, b2);
            }
        }
    }
    const int v0 = max(first, v_first);
    if (!E4M3) {
        if (on)
            for (int which = v0; which < last; which++) {
                load(a.qkv + row * a.stride + o, which);
                bf16 *to = wide_row(place, which - v_first, 1);
                *reinterpret_cast<uint4 *>(to + o) = raw1;
                *reinterpret_cast<uint4 *>(to + HALF + o) = raw2;
            }
        return;
    }
    auto value = [&](long long from, int which, uint8_t *page, int j, uint8_t *b1, uint8_t *b2) { /* a row's bytes and scale */
        float x1[VEC], x2[VEC];
        unpack_bf16x8(raw1, x1);
        unpack_bf16x8(raw2, x2);
        if (which + 1 < last) load(a.qkv + from * a.stride + o, which + 1);
        const float scale = quantise(x1, x2, b1, b2);
        if (t == 0) reinterpret_cast<float *>(page + PAGE_VS)[j] = scale;
    };
    if (start >= 0 && v0 < last) { /* the run that begins here */
        const long long from = row + start;
        const int at = near_place[BACK + start + g], j = at % PAGE_TOKENS;
        load(a.qkv + from * a.stride + o, v0);
        for (int which = v0; which < last; which++) {
            uint8_t b1[VEC], b2[VEC], *page = page_of(at, which - v_first);
            value(from, which, page, j, b1, b2);
            /* word k of dim d sits at word k ^ ((d >> 3) & 3): the eight lanes of a row are not all on one bank */
            const int col = g ^ ((t & 3) << 2);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                vt[o + i][col] = b1[i];
                vt[HALF + o + i][col] = b2[i];
            }
            __syncthreads();
            const int d = threadIdx.x, sw = (d >> 3) & 3;
            const uint32_t *w = reinterpret_cast<const uint32_t *>(vt[d]);
            *reinterpret_cast<uint4 *>(page + page_v_byte(j - g, d)) = make_uint4(w[sw], w[1 ^ sw], w[2 ^ sw], w[3 ^ sw]);
            __syncthreads(); /* the next v head row reuses the tile */
        }
    }
    if (on && !grouped && v0 < last) { /* rows by themselves */
        load(a.qkv + row * a.stride + o, v0);
        for (int which = v0; which < last; which++) {
            uint8_t b1[VEC], b2[VEC], *page = page_of(place, which - v_first);
            value(row, which, page, place % PAGE_TOKENS, b1, b2);
            store_v_row(page, place % PAGE_TOKENS, t, b1, b2);
        }
    }
}

} /* namespace */

extern "C" int paged_append(const void *qkv, const void *q_gain, const void *k_gain, const void *cos, const void *sin, const void *pos,
                            const void *place, void *q_out, void *pool, long long rows, int Hq, int Hkv, long long qkv_row_stride, int table_len,
                            int n_pages, int e4m3, void *status, void *stream) {
    if (rows < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || table_len <= 0 || n_pages <= 0 || n_pages > 0x7fffffff / PAGE_TOKENS) return NCB_ERR_ARG;
    if (qkv_row_stride < (long long)(Hq + 2ll * Hkv) * HEAD_DIM) return NCB_ERR_ARG;
    if (rows == 0) return NCB_OK;
    if (!qkv || !q_gain || !k_gain || !cos || !sin || !pos || !place || !q_out || !pool) return NCB_ERR_ARG;
    const uintptr_t all = (uintptr_t)qkv | (uintptr_t)q_gain | (uintptr_t)k_gain | (uintptr_t)cos | (uintptr_t)sin | (uintptr_t)q_out | (uintptr_t)pool;
    if (all % 16 || qkv_row_stride % 8) return NCB_ERR_ALIGN;
    const long long blocks = (rows + ROWS_PER_BLOCK - 1) / ROWS_PER_BLOCK;
    const int heads = Hq + 2 * Hkv;
    if (blocks > 0x7fffffffll || heads > 65535) return NCB_ERR_ARG;
    /* decode steps: one head row per block; large passes: up to 8 as long as about 2,048 blocks remain */
    long long per = blocks * heads / 2048;
    per = per < 1 ? 1 : per > 8 ? 8 : per;
    const AppendArgs a = {(const bf16 *)qkv, (const float *)q_gain, (const float *)k_gain, (const float *)cos, (const float *)sin,
                          (const int32_t *)pos, (const int32_t *)place, (bf16 *)q_out, (uint8_t *)pool, rows, qkv_row_stride, Hq, Hkv, table_len,
                          n_pages, (int)per, (int *)status};
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)blocks, (unsigned)((heads + per - 1) / per));
    config.blockDim = dim3(BLOCK);
    config.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, e4m3 ? k_paged_append<true> : k_paged_append<false>, a) == cudaSuccess ? NCB_OK : NCB_ERR_LAUNCH;
}
