/*
 * Shared by page_plan.cu and paged_attn.cu: the schedule of a paged attention call. Work is cut into owners: consecutive new rows of one request
 * which, with all query heads of a key/value head (query slots), one block can take. Requests of at most SMALL_SLOTS query slots belong to the small kernel,
 * the others to the tile kernel; each class has a schedule of its own.
 *
 * An owner weighs its pages and OVERHEAD (what a block spends on it besides); `before` are the exclusive sums of the weights, `total` their sum. The work of all
 * key/value heads, one after the other, is a line of length total * heads, and block b has the piece [b * share, (b + 1) * share) of it, wherever owners
 * begin and end: every block has the same to do, whatever the lengths are. A block leaves at most two owners unfinished, the one that it goes on with
 * from the block before it and the one that the next block goes on with: their states go to parts 2 b and 2 b + 1, and the schedule lists which
 * parts are joined. Where the blocks would not be done much later with whole owners, from the last (a request's longest) on, or where small owners have few pages at most, none is cut:
 * each is a block's, and no state is written or read.
 */
#pragma once

#include "ncb_common.cuh"

namespace {
namespace paged {

constexpr int SMALL_SLOTS = 16, TILE_SLOTS = 256; /* query slots of a block of the small kernel, of the tile kernel (two tiles of 128) */
constexpr int MAX_GROUP = 64;                     /* query heads per key/value head */
constexpr int HEADER_WORDS = 8;                   /* owners, total, share, whole: of a class */
constexpr int OWNER_WORDS = 8, START_WORDS = 4, PIECE_WORDS = 8, JOIN_WORDS = 8;
constexpr int WHOLE_ROUNDS = 8; /* tiles are cut only where there are fewer than this many for every block */
/* Small owners are cut only where a request may have more pages than this: the launch that joins states costs more than it saves (three users of up to 11 pages, 10 heads:
 * 8.7 us whole, 12.4 cut; the host needs a launch and a workspace less). */
constexpr int WHOLE_WIDTH = 16;
/* What cutting owners costs a block, in pages: an overhead more, and the states. Small owners and few rows (33 requests of 5 behind a window of 512, 16 heads over 4: 34.0 us cut,
 * 31.7 whole; of 2,048: 55.5, 62; 100 of one row, 2,000 positions: 43.4, 41.5); full tiles (bf16, 16 heads over 4: prompts of 2,500, 4,096 and 6,000 rows 54.8, 101 and 179 us cut, 50.8, 78
 * and 154 whole; eight of 512 behind 4,000 positions, 32 over 8, e4m3, whose last round would be half empty: 398, 426; a mixed step 91, 126). */
constexpr int SMALL_SLACK = 6, FEW_SLACK = 8, TILE_SLACK = 20;

struct alignas(16) Owner {
    int request, row, rows; /* absolute first row */
    int pos;                /* position of the first row */
    int page0, pages;       /* pages of the request that its rows see; no pages: rows that are not served, to become zeros */
    int before;             /* weights of the owners before it */
    int pad;
};
/* Where a block's part of the line begins. */
struct alignas(16) Start {
    int owner, head;
    int local; /* place within the owner, whose overhead comes first */
    int piece; /* tiles: the block's first piece; the next block's is behind its last */
};
/* A block's share of an owner, ready for the tile kernel. */
struct Piece {
    int request, row, rows, pos; /* as the owner's */
    int page0, pages;            /* of the request */
    int head;
    int part; /* where the state goes; -1: it is the whole owner, and the block writes its rows */
};
/* What k_paged_merge does at the end of a block's part of the line where an owner is cut for the first time: its states are part 2 first + 1 and parts
 * 2 b of the blocks b behind. */
struct Join {
    int row, slots, head; /* the owner's first row; its query slots; none: nothing to do */
    int first, last;      /* blocks */
    int pad[3];
};
static_assert(sizeof(Join) == 4 * JOIN_WORDS && sizeof(Owner) == 4 * OWNER_WORDS && sizeof(Start) == 4 * START_WORDS && sizeof(Piece) == 4 * PIECE_WORDS, "schedule layout");

struct Class {
    long long owners; /* at most */
    int rows_per, slots; /* of an owner */
    int blocks, overhead, least; /* blocks that run at once; weight of an owner besides its pages; least share */
    int slack;                   /* what an owner may weigh above a block's share and still not be cut */
};
struct Caps {
    Class small, tile;
    int smalls, tiles; /* whether the kernel has anything. Without tiles the small kernel also has what is too long and only gets zeros. */
};
/* `blocks`: SMs; three blocks of the small kernel run on each, one of the tile kernel. */
static __host__ __device__ __forceinline__ Caps caps_of(int requests, long long rows, int max_fresh, int group, int blocks) {
    Caps c = {};
    const long long one_each = requests < rows ? requests : rows;
    const int few = SMALL_SLOTS / group; /* 0: even one row has too many slots */
    c.smalls = few > 0 && rows > 0, c.tiles = max_fresh > few && rows > few;
    if (c.smalls) {
        /* Without tiles, rows of requests that are not served, however many, are in owners of no more slots than the others', which the kernel is chosen for. */
        const int per = max_fresh < few ? max_fresh : few;
        c.small.rows_per = per;
        c.small.slots = per * group;
        c.small.owners = c.tiles ? one_each : (rows + one_each * (per - 1)) / per;
        c.small.blocks = 3 * blocks, c.small.overhead = 2, c.small.least = 6, c.small.slack = SMALL_SLACK;
    }
    if (c.tiles) {
        const long long longer = rows / (few + 1); /* requests that have tiles */
        c.tile.rows_per = TILE_SLOTS / 2 / group * 2;
        c.tile.slots = (max_fresh < c.tile.rows_per ? max_fresh : c.tile.rows_per) * group;
        c.tile.owners = rows / c.tile.rows_per + (longer < one_each ? longer : one_each);
        c.tile.blocks = blocks, c.tile.overhead = 4, c.tile.least = 8, c.tile.slack = max_fresh <= c.tile.rows_per / 2 ? FEW_SLACK : TILE_SLACK;
    }
    return c;
}
/* A class in a schedule: header, owners, starts (of one block more than there are), joins (one per block), for tiles the pieces: one per owner and head and one per cut. */
static __host__ __device__ __forceinline__ long long starts_at(const Class &c) { return HEADER_WORDS + c.owners * OWNER_WORDS; }
static __host__ __device__ __forceinline__ long long joins_at(const Class &c) { return starts_at(c) + (c.blocks + 2) / 2 * 2 * START_WORDS; }
static __host__ __device__ __forceinline__ long long pieces_at(const Class &c) { return joins_at(c) + (long long)c.blocks * JOIN_WORDS; }
static __host__ __device__ __forceinline__ long long class_words(const Class &c, bool tile) {
    return c.owners ? pieces_at(c) + (tile ? (WHOLE_ROUNDS + 1ll) * c.blocks * PIECE_WORDS : 0) : 0;
}
static __host__ __device__ __forceinline__ long long schedule_words(const Caps &c) { return class_words(c.small, false) + class_words(c.tile, true); }
static __host__ __device__ __forceinline__ long long class_at(const Caps &c, int tile) { return tile ? class_words(c.small, false) : 0; }
/* Floats of the workspace: two parts per block of each class. */
static __host__ __device__ __forceinline__ long long parts_at(const Caps &c, int tile) { return tile ? 2ll * c.small.blocks * c.small.slots * PART : 0; }
static __host__ __device__ __forceinline__ long long workspace_floats(const Caps &c) { return parts_at(c, 1) + 2ll * c.tile.blocks * c.tile.slots * PART; }

static __host__ __forceinline__ bool sizes_ok(int requests, long long rows, int max_fresh, int group, int kv_heads, int blocks) {
    return requests > 0 && requests <= NCB_PLAN_REQUESTS && rows >= 0 && rows <= (1ll << 26) && max_fresh > 0 && group > 0 && group <= MAX_GROUP &&
           kv_heads > 0 && kv_heads <= 65535 && blocks > 0 && blocks <= (1 << 16);
}

struct PagedArgs { /* of paged_attn's kernels */
    ncb_paged p;
    Caps caps;
    float scale_log2;
};

/* A record of the schedule, not through L1. */
template <typename Record> __device__ __forceinline__ Record of_l2(const Record *from) {
    static_assert(sizeof(Record) % 16 == 0, "in vectors");
    Record to;
#pragma unroll
    for (int i = 0; i < (int)sizeof(Record) / 16; i++) reinterpret_cast<int4 *>(&to)[i] = __ldcg(reinterpret_cast<const int4 *>(from) + i);
    return to;
}

/* A class's schedule as kernels read it. */
struct Line {
    const Owner *owners;
    const Start *starts;
    const Piece *pieces;
    int n, heads, overhead;
    long long total, share; /* of one key/value head; of a block */
    bool whole;

    __device__ __forceinline__ Line(const PagedArgs &args, int tile) {
        const Class &c = tile ? args.caps.tile : args.caps.small;
        const int *w = args.p.work + class_at(args.caps, tile);
        const int4 header = of_l2(reinterpret_cast<const int4 *>(w));
        owners = reinterpret_cast<const Owner *>(w + HEADER_WORDS);
        starts = reinterpret_cast<const Start *>(w + starts_at(c));
        pieces = reinterpret_cast<const Piece *>(w + pieces_at(c));
        n = header.x, total = header.y, share = header.z, whole = header.w != 0;
        heads = args.p.Hkv, overhead = c.overhead;
    }
    __device__ __forceinline__ long long all() const { return total * heads; }
};

/* What a block of a class that is cut does, one piece after the other. */
struct Walk {
    Owner o;
    int head, page0, page1; /* the piece: pages [page0, page1) of the owner's, for this key/value head */
    int part;               /* as Piece's */

    /* From `start` on, `left` of the line. */
    __device__ __forceinline__ Walk(const Owner *owners, int n, int overhead, const Start &start, int left, int block)
        : owners(owners), n(n), overhead(overhead), at(start.owner), next_head(start.head), local(start.local), left(left), block(block) {}
    /* The next piece; false at the end. */
    __device__ __forceinline__ bool next() {
        while (left > 0) {
            o = of_l2(owners + at), head = next_head;
            const int pages = max(o.pages, 1), from = max(local - overhead, 0), to = min(local + left - overhead, pages);
            const int used = overhead + pages - local; /* to the owner's end */
            part = from == 0 && to == pages ? -1 : 2 * block + (from == 0);
            page0 = from, page1 = min(to, o.pages);
            left -= used, local = 0;
            if (++at == n) at = 0, next_head++;
            if (from < to) return true; /* else only (some of) its overhead lies here */
        }
        return false;
    }

private:
    const Owner *owners;
    int n, overhead, at, next_head, local, left, block;
};

} /* namespace paged */
} /* namespace */
