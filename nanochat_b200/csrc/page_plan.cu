/*
 * page_plan: block tables, positions and places of one step from the requests' lengths, on the GPU, so that a captured step serves
 * lengths that change; page_release: finished requests give their pages back; page_trim: requests whose lengths go back (rejected drafts) give back the
 * pages behind them. No counterpart in the reference, whose slots are of
 * one size (inference/decoder.py:112-121).
 *
 * Every block repeats the same two prefix sums over the requests (rows, then new pages) in shared memory, 16 KB for a thousand requests,
 * instead of waiting for a launch that makes them once; then the row blocks write rows and table entries, each finding its
 * request by a binary search in the sums, and one block per window and class makes a schedule of the attention's work (paged.cuh). A step's bytes
 * are a few per row, so the launch is bound by latency: the chain of sums and searches. 64 requests 8 to 10 us, 1,025 requests 12 to 15.
 */
#include <atomic>

#include "paged.cuh"

namespace {

using namespace paged;

constexpr int THREADS = 1024, WARPS = THREADS / 32;

/* Exclusive prefix sum of v over the block's threads; *total gets the sum. */
__device__ __forceinline__ long long block_sum_before(long long v, long long *sums, long long *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    __syncthreads(); /* the sums of the call before have been read */
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    long long w = sums[lane]; /* every warp sums the warps' sums for itself: no third barrier */
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += x;
    }
    *total = __shfl_sync(0xffffffffu, w, 31);
    const long long before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    return (warp > 0 ? before : 0) + upto - v;
}

/* The first index whose value is greater than x in an ascending array. */
__device__ __forceinline__ int first_above(const int *a, int n, int x) {
    int low = 0, high = n;
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (a[mid] > x) high = mid;
        else low = mid + 1;
    }
    return low;
}

__device__ __forceinline__ int pages_for(long long positions) { return (int)((positions + PAGE_TOKENS - 1) / PAGE_TOKENS); }
__device__ __forceinline__ int clamp_int(long long v) { return v > 0x7fffffffll ? 0x7fffffff : (int)v; }

struct Requests { /* shared memory, one value a request each */
    int *row_end, *page_end; /* inclusive sums of rows and of new pages */
    int *cached, *served;    /* served: rows, 0 for a request that is not */
    int *owner_end;          /* schedule blocks: inclusive sum of owners */
};
constexpr int REQUEST_BYTES = 5 * 4;

/* How long the last block has work if owners are whole: no less than the heaviest, nor than what some block has of the n heaviest, ceil(n * heads / blocks) of them
 * at least, for n down to each of sixteen weights; and hardly more, a request's heaviest going first. (All sorted by weight is slower, eight prompts of 600 rows 48 us
 * for 45: neighbours no longer read the same pages.) heaviest: of the thread's owners, which it has written itself. */
__device__ long long longest_whole(const Owner *records, int owners, int heads, const Class &c, int heaviest) {
    constexpr int STEPS = 16;
    __shared__ int most, count[STEPS], least[STEPS];
    const int tid = threadIdx.x;
    if (tid == 0) most = 1;
    if (tid < STEPS) count[tid] = 0, least[tid] = 0x7fffffff;
    __syncthreads();
    heaviest = __reduce_max_sync(0xffffffffu, heaviest);
    if (tid % 32 == 0) atomicMax(&most, heaviest);
    __syncthreads();
    const int top = most;
    for (int o = tid; o < owners; o += THREADS) {
        const int weight = max(records[o].pages, 1) + c.overhead, step = ((long long)weight * STEPS - 1) / top;
        atomicAdd(count + step, 1);
        atomicMin(least + step, weight);
    }
    __syncthreads();
    long long last = top, n = 0;
#pragma unroll 1
    for (int i = STEPS - 1; i >= 0; i--)
        if (count[i]) n += count[i], last = max(last, (n * heads + c.blocks - 1) / c.blocks * least[i]);
    return last;
}

/* The schedule of one window's attention, of one class of requests (paged.cuh). */
__device__ void schedule(const ncb_page_plan &a, const Requests &r, int window, int tile, int *work, long long *sums) {
    const Caps caps = caps_of(a.requests, a.rows, a.max_fresh, a.group, a.blocks);
    const Class &c = tile ? caps.tile : caps.small;
    const int tid = threadIdx.x, per = (a.requests + THREADS - 1) / THREADS, b0 = tid * per, b1 = min(b0 + per, a.requests);
    const int rows_per = c.rows_per, rows = (int)a.rows, few = SMALL_SLOTS / a.group;
    auto rows_of = [&](int b) { /* not served ones among them: zeros to write */
        const int n = min(r.row_end[b], rows) - min(b ? r.row_end[b - 1] : 0, rows);
        return caps.tiles && (n > few) != (tile != 0) ? 0 : n;
    };
    long long total, mine = 0;
    for (int b = b0; b < b1; b++) mine += (rows_of(b) + rows_per - 1) / rows_per;
    long long at = block_sum_before(mine, sums, &total);
    for (int b = b0; b < b1; b++) r.owner_end[b] = (int)(at += (rows_of(b) + rows_per - 1) / rows_per);
    __syncthreads();
    const int owners = (int)min(total, c.owners);
    work += class_at(caps, tile);
    Owner *records = reinterpret_cast<Owner *>(work + HEADER_WORDS);
    int *before = r.page_end; /* the sums once more, for the searches below (nobody reads the pages' in this block) */
    long long weight = 0;
    int heaviest = 0;
    for (int from = 0; from < owners; from += THREADS) {
        const int o = from + tid;
        Owner w = {};
        if (o < owners) {
            w.request = first_above(r.owner_end, a.requests, o);
            const int row0 = (o - (w.request ? r.owner_end[w.request - 1] : 0)) * rows_per;
            w.row = (w.request ? r.row_end[w.request - 1] : 0) + row0;
            w.rows = min(rows_per, rows_of(w.request) - row0);
            if (r.served[w.request] > 0) {
                w.pos = r.cached[w.request] + row0;
                w.page0 = window > 0 && w.pos + 1 > window ? (w.pos + 1 - window) / PAGE_TOKENS : 0;
                w.pages = (w.pos + w.rows - 1) / PAGE_TOKENS + 1 - w.page0;
            }
        }
        const long long sum = weight + block_sum_before(o < owners ? max(w.pages, 1) + c.overhead : 0, sums, &total);
        if (o < owners) {
            w.before = (int)sum;
            records[o] = w;
            if (o < a.requests) before[o] = w.before;
            heaviest = max(heaviest, max(w.pages, 1) + c.overhead);
        }
        weight += total;
    }
    const long long all = weight * a.kv_heads, share = min(max((all + c.blocks - 1) / c.blocks, (long long)c.least), 0x7fffffffll);
    const long long each = (long long)owners * a.kv_heads;
    bool whole = tile ? each >= (long long)WHOLE_ROUNDS * c.blocks : a.width <= WHOLE_WIDTH;
    if (!whole && (tile || each <= c.blocks)) { /* small owners have a block each, or are cut */
        const long long last = longest_whole(records, owners, a.kv_heads, c, heaviest);
        whole = last <= share + c.slack;
    }
    if (tid == 0) *reinterpret_cast<int4 *>(work) = make_int4(owners, (int)weight, (int)share, whole);
    Join *joins = reinterpret_cast<Join *>(work + joins_at(c));
    if (whole || owners == 0) {
        for (int b = tid; b < c.blocks; b += THREADS) joins[b].slots = 0;
        return;
    }
    __syncthreads();
    Start *starts = reinterpret_cast<Start *>(work + starts_at(c));
    Piece *pieces = reinterpret_cast<Piece *>(work + pieces_at(c));
    const bool listed = owners <= a.requests;
    long long count = 0; /* of pieces */
    for (int from = 0; from <= c.blocks; from += THREADS) {
        const int b = from + tid;
        const long long x = b * share;
        const bool on = b <= c.blocks && x < all;
        Start start = {0, 0, 0, 0};
        if (on) {
            start.head = (int)(x / weight);
            const int place = (int)(x - start.head * weight);
            int low = 0, high = owners; /* the last owner whose `before` is at most `place` */
            while (high - low > 1) {
                const int mid = (low + high) >> 1;
                if ((listed ? before[mid] : records[mid].before) <= place) low = mid;
                else high = mid;
            }
            start.owner = low, start.local = place - (listed ? before[low] : records[low].before);
        }
        if (tile) { /* the block's pieces: counted, then written */
            int mine = 0;
            if (on)
                for (Walk walk(records, owners, c.overhead, start, (int)min(share, all - x), b); walk.next();) mine++;
            const long long to = count + block_sum_before(mine, sums, &total);
            start.piece = (int)to;
            if (on) {
                int i = 0;
                for (Walk walk(records, owners, c.overhead, start, (int)min(share, all - x), b); walk.next() && to + i < (WHOLE_ROUNDS + 1ll) * c.blocks; i++)
                    pieces[to + i] = Piece{walk.o.request, walk.o.row, walk.o.rows, walk.o.pos, walk.o.page0 + walk.page0, walk.page1 - walk.page0, walk.head, walk.part};
            }
            count += total;
        }
        if (b <= c.blocks) starts[b] = start;
        if (b > 0 && b <= c.blocks) { /* an owner that this block goes on with, the block before having begun with it? */
            Join join = {};
            if (on && start.local > c.overhead) {
                const Owner &o = records[start.owner];
                const long long begin = start.head * weight + (listed ? before[start.owner] : o.before) + c.overhead;
                const int first = (int)(begin / share), end = (int)((begin + max(o.pages, 1) - 1) / share);
                if (first == b - 1) join = Join{o.row, o.rows * a.group, start.head, first, end, {}};
            }
            joins[b - 1] = join;
        }
    }
}

struct PlanArgs {
    ncb_page_plan p;
    int row_blocks, first_class; /* 1: only tiles */
    long long words;
};

__global__ void __launch_bounds__(THREADS) k_page_plan(const PlanArgs args) {
    extern __shared__ __align__(16) int smem[];
    __shared__ long long sums[WARPS];
    __shared__ int last;
    const ncb_page_plan &a = args.p;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, n = a.requests, per = (n + THREADS - 1) / THREADS, b0 = tid * per, end = min(b0 + per, n);
    const Requests r = {smem, smem + n, smem + 2 * n, smem + 3 * n, smem + 4 * n};
    const int free_count = max(0, min(*reinterpret_cast<const volatile int *>(a.free_count), a.n_pages));
    for (int b = tid; b < n; b += THREADS) r.cached[b] = a.cached[b], r.served[b] = a.fresh[b];
    __syncthreads();
    long long total, mine = 0;
    for (int b = b0; b < end; b++) mine += max(r.served[b], 0);
    long long at = block_sum_before(mine, sums, &total);
    const int rows_used = clamp_int(min(total, a.rows));
    bool bad = false;
    mine = 0;
    for (int b = b0; b < end; b++) {
        const int cached = r.cached[b], fresh = r.served[b];
        at += max(fresh, 0);
        r.row_end[b] = clamp_int(at);
        const bool ok = cached >= 0 && fresh >= 0 && fresh <= a.max_fresh && (long long)cached + fresh <= (long long)a.width * PAGE_TOKENS && (fresh == 0 || at <= a.rows);
        bad |= !ok;
        if (!ok || fresh == 0) r.served[b] = 0;
        else mine += pages_for((long long)cached + fresh) - pages_for(cached);
    }
    long long new_pages;
    at = block_sum_before(mine, sums, &new_pages);
    bool none = false;
    mine = 0; /* pages that are taken */
    for (int b = b0; b < end; b++) {
        const int fresh = r.served[b], need = fresh > 0 ? pages_for((long long)r.cached[b] + fresh) - pages_for(r.cached[b]) : 0;
        at += need;
        r.page_end[b] = clamp_int(at);
        if (need > 0 && at > free_count) r.served[b] = 0, none = true;
        else mine += need;
    }
    long long taken;
    block_sum_before(mine, sums, &taken); /* its barriers publish the arrays */
    if (blockIdx.x >= args.row_blocks) {
        const int w = (blockIdx.x - args.row_blocks) % a.n_windows, tile = (blockIdx.x - args.row_blocks) / a.n_windows + args.first_class;
        schedule(a, r, a.windows[w], tile, a.work + w * args.words, sums);
    } else {
        if (blockIdx.x == 0) {
            if (bad) flag(a.status, NCB_DEV_BAD_LENGTH);
            if (none) flag(a.status, NCB_DEV_NO_PAGES);
            for (int b = tid; b < n; b += THREADS) {
                a.row_start[b + 1] = r.row_end[b];
                a.served[b] = r.served[b];
            }
            if (tid == 0) a.row_start[0] = 0;
        }
        /* page i of request b's new ones; i and b must be in range */
        auto new_page = [&](int b, int i) {
            const int before = b ? r.page_end[b - 1] : 0, from = free_count - 1 - before - i;
            const int page = from >= 0 ? a.free_pages[from] : -1;
            if ((unsigned)page < (unsigned)a.n_pages) return page;
            flag(a.status, NCB_DEV_BAD_PAGE);
            return -1;
        };
        const int step = args.row_blocks * THREADS, first = blockIdx.x * THREADS + tid;
        for (long long i = first; i < min(new_pages, (long long)free_count); i += step) {
            const int b = first_above(r.page_end, n, (int)i);
            if (r.served[b] == 0) continue;
            const int before = b ? r.page_end[b - 1] : 0, j = (int)i - before;
            a.table[(size_t)b * a.width + pages_for(r.cached[b]) + j] = new_page(b, j);
        }
        for (long long row = first; row < a.rows; row += step) {
            int pos = -1, place = -1, request = -1;
            if (row < rows_used) {
                request = first_above(r.row_end, n, (int)row);
                if (r.served[request] > 0) {
                    const int cached = r.cached[request], have = pages_for(cached);
                    pos = cached + (int)row - (request ? r.row_end[request - 1] : 0);
                    const int p = pos / PAGE_TOKENS;
                    int page;
                    if (p < have) {
                        page = a.table[(size_t)request * a.width + p];
                        if ((unsigned)page >= (unsigned)a.n_pages) flag(a.status, NCB_DEV_BAD_PAGE), page = -1;
                    } else {
                        page = new_page(request, p - have);
                    }
                    if (page >= 0) place = page * PAGE_TOKENS + pos % PAGE_TOKENS;
                }
            }
            a.pos[row] = pos, a.place[row] = place, a.request[row] = request;
        }
    }
    /* what may be written over its input (lens over cached, free_left over free_count) is left to the last block: all have read by then */
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        last = atomicAdd(a.ticket, 1) == (int)gridDim.x - 1;
        if (last) {
            *a.free_left = free_count - (int)taken;
            *a.ticket = 0;
        }
    }
    __syncthreads();
    if (last)
        for (int b = tid; b < n; b += THREADS) a.lens[b] = max(r.cached[b], 0) + r.served[b];
}

struct ReleaseArgs {
    int *table, *lens;
    const int *release, *keep; /* one of them: requests that keep nothing; positions that each keeps */
    int *free_pages, *free_count;
    int requests, width, n_pages;
    int *status;
};

/* One block: requests in order, a request's pages from its last to its first, so that the next request gets them in order again. A turn of 32 requests waits for the
 * sum of their pages, 1.1 to 2.4 us: all of 64 requests of up to 128 pages 13 us, of 1,025 of up to 64 pages 81, of 8,192 of up to 16 pages 499; five positions less each 9, 54, 380. */
__global__ void __launch_bounds__(THREADS) k_page_release(const ReleaseArgs a) {
    __shared__ long long sums[WARPS];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long count = max(0, min(*a.free_count, a.n_pages));
    auto valid = [&](int page) { return (unsigned)page < (unsigned)a.n_pages; };
    for (int from = 0; from < a.requests; from += WARPS) { /* a warp per request: its entries are counted, then moved */
        const int b = from + warp;
        const bool on = b < a.requests && (a.keep || a.release[b] != 0);
        const int had = on ? max(a.lens[b], 0) : 0, keep = on && a.keep ? a.keep[b] : 0, stay = keep < 0 ? had : min(keep, had);
        if (keep < 0 && lane == 0) flag(a.status, NCB_DEV_BAD_LENGTH);
        const int held = min(pages_for(had), a.width), first = min(pages_for(stay), held);
        int *entries = a.table + (size_t)(on ? b : 0) * a.width;
        int good = 0;
        for (int i = first; i < held; i += 32) {
            const bool in = i + lane < held, ok = in && valid(entries[i + lane]);
            good += __popc(__ballot_sync(0xffffffffu, ok));
            if (in && !ok) flag(a.status, NCB_DEV_BAD_PAGE);
        }
        long long total;
        long long at = count + block_sum_before(lane == 0 ? good : 0, sums, &total);
        at = __shfl_sync(0xffffffffu, at, 0) + good; /* the end of this request's pages in the list */
        for (int i = first; i < held; i += 32) {
            const int page = i + lane < held ? entries[i + lane] : -1;
            const uint32_t ok = __ballot_sync(0xffffffffu, valid(page));
            if (valid(page)) {
                const long long to = at - 1 - __popc(ok & ((1u << lane) - 1u));
                if (to < a.n_pages) a.free_pages[to] = page;
                else flag(a.status, NCB_DEV_BAD_PAGE); /* more pages than the pool has: some came back twice */
            }
            at -= __popc(ok);
            if (i + lane < held) entries[i + lane] = -1;
        }
        if (on && lane == 0) a.lens[b] = stay;
        count += total;
    }
    __syncthreads();
    if (tid == 0) *a.free_count = (int)min(count, (long long)a.n_pages);
}

/* Opts k_page_plan in to the arrays of the most requests, once per device and whatever the call's size: what a launch may have without is 48 KB for
 * these and the kernel's own shared memory together. */
cudaError_t allow_requests() {
    static std::atomic<unsigned long long> ready{0};
    int device;
    cudaError_t rc = cudaGetDevice(&device);
    if (rc != cudaSuccess) return rc;
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (ready.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    rc = cudaFuncSetAttribute(k_page_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, REQUEST_BYTES * NCB_PLAN_REQUESTS);
    if (rc == cudaSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
    return rc;
}

cudaError_t launch(void (*kernel)(const PlanArgs), int grid, int smem, cudaStream_t stream, const PlanArgs &args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args);
}

int give_back(const ReleaseArgs &a, void *stream) {
    if (a.requests <= 0 || a.requests > NCB_PLAN_REQUESTS || a.width <= 0 || a.n_pages <= 0) return NCB_ERR_ARG;
    if (!a.table || !a.lens || (!a.release && !a.keep) || !a.free_pages || !a.free_count) return NCB_ERR_ARG;
    k_page_release<<<1, THREADS, 0, (cudaStream_t)stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? NCB_OK : NCB_ERR_LAUNCH;
}

} /* namespace */

extern "C" {

long long page_plan_words(int requests, long long rows, int max_fresh, int group, int kv_heads, int blocks) {
    if (!sizes_ok(requests, rows, max_fresh, group, kv_heads, blocks)) return -1;
    return schedule_words(caps_of(requests, rows, max_fresh, group, blocks));
}

int page_plan(const ncb_page_plan *args, void *stream) {
    if (!args) return NCB_ERR_ARG;
    const ncb_page_plan &a = *args;
    if (!sizes_ok(a.requests, a.rows, a.max_fresh, a.group, a.kv_heads, a.blocks)) return NCB_ERR_ARG;
    if (a.width <= 0 || a.width > (1 << 16) || a.n_pages <= 0 || a.n_pages > 0x7fffffff / PAGE_TOKENS || a.n_windows < 0 || a.n_windows > NCB_PLAN_WINDOWS) return NCB_ERR_ARG;
    for (int w = 0; w < a.n_windows; w++)
        if (a.windows[w] < 0) return NCB_ERR_ARG;
    if (!a.table || !a.cached || !a.fresh || !a.free_pages || !a.free_count || !a.free_left || !a.row_start || !a.served || !a.lens || !a.ticket ||
        (a.rows > 0 && (!a.pos || !a.place || !a.request)) || (a.n_windows > 0 && !a.work))
        return NCB_ERR_ARG;
    if ((uintptr_t)a.work % 16) return NCB_ERR_ALIGN;
    const Caps caps = caps_of(a.requests, a.rows, a.max_fresh, a.group, a.blocks);
    PlanArgs p = {a, 1, !caps.smalls, schedule_words(caps)};
    /* a block writes 2,048 rows in about the time that its sums take; more blocks than SMs would repeat them */
    p.row_blocks = (int)((a.rows + 2047) / 2048);
    p.row_blocks = p.row_blocks < 1 ? 1 : p.row_blocks > 64 ? 64 : p.row_blocks;
    if (allow_requests() != cudaSuccess) return NCB_ERR_LAUNCH;
    return launch(k_page_plan, p.row_blocks + a.n_windows * (caps.smalls + caps.tiles), REQUEST_BYTES * a.requests, (cudaStream_t)stream, p) == cudaSuccess ? NCB_OK : NCB_ERR_LAUNCH;
}

int page_release(int *table, int *lens, const int *release, int *free_pages, int *free_count, int requests, int width, int n_pages, int *status,
                 void *stream) {
    return give_back({table, lens, release, nullptr, free_pages, free_count, requests, width, n_pages, status}, stream);
}

int page_trim(int *table, int *lens, const int *keep, int *free_pages, int *free_count, int requests, int width, int n_pages, int *status, void *stream) {
    return give_back({table, lens, nullptr, keep, free_pages, free_count, requests, width, n_pages, status}, stream);
}

} /* extern "C" */
