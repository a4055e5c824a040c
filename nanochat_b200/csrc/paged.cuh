/*
 * Shared by page_plan.cu and paged_attn.cu: what the schedule of a paged attention call looks like in memory, and how much of it
 * there can be. Work is cut into owners: the `rows_per` consecutive new rows of one request (with all query heads of a key/value head:
 * query slots) that one block takes; an owner's pages are cut into chunks of at most a chosen number of pages. An owner of several chunks leaves
 * a state per chunk in the workspace and is listed for the merge.
 */
#pragma once

#include "ncb_common.cuh"

namespace {
namespace paged {

constexpr int SMALL_SLOTS = 16, TILE_SLOTS = 128; /* query slots of a block of the small kernel, of the tile kernel */
constexpr int MAX_GROUP = 64;                     /* query heads per key/value head */
constexpr int TILE_WAVES = 2;                     /* cut tiles are at most this often what runs at once */
constexpr int HEADER_WORDS = 16;                  /* entries and merges of the small kernel, of the tile kernel */
constexpr int ENTRY_WORDS = 8, MERGE_WORDS = 4;

struct Entry { /* one block's work, for each key/value head */
    int request, row0, rows;  /* rows row0 .. of the request's new rows */
    int page0, page1;         /* pages of the request */
    int part;                 /* where its state goes; -1: the block normalises and writes its rows itself */
    int pad[2];
};
struct Merge { /* an owner of several chunks */
    int row, rows; /* absolute rows */
    int part, parts;
};
static_assert(sizeof(Entry) == 4 * ENTRY_WORDS && sizeof(Merge) == 4 * MERGE_WORDS, "schedule layout");

/* How many entries a schedule may aim at: every key/value head runs each of them. */
static __host__ __device__ __forceinline__ int units_of(int blocks, int kv_heads) { return blocks / kv_heads > 1 ? blocks / kv_heads : 1; }

static __host__ __device__ __forceinline__ int small_blocks(int blocks) { return blocks / 2 * 3; } /* three per SM instead of two */

/* Bounds of a schedule, and where its parts lie. The tile kernel has the requests of more than SMALL_SLOTS query slots, the small kernel the
 * others; where no request may have so many, no tile kernel runs, and the small kernel also has what is too long and only gets zeros.
 * A chunk of the small kernel is at least total / (waves * units) pages: the owners that are cut are at most waves * units, their
 * chunks at most twice that. Tiles are cut only where all entries are then at most TILE_WAVES * units. */
struct Class {
    long long owners, entries, merges, parts;
    int rows_per, slots; /* of an owner */
    int units, waves;
};
struct Caps {
    Class small, tile;
    int smalls, tiles; /* whether the kernel has anything */
};
static __host__ __device__ __forceinline__ Caps caps_of(int requests, long long rows, int max_fresh, int group, int kv_heads, int blocks) {
    Caps c = {};
    const long long one_each = requests < rows ? requests : rows;
    const int few = SMALL_SLOTS / group; /* 0: even one row has too many slots */
    c.smalls = few > 0, c.tiles = max_fresh > few;
    if (c.smalls) {
        c.small.rows_per = few;
        c.small.slots = (max_fresh < few ? max_fresh : few) * group;
        c.small.units = units_of(small_blocks(blocks), kv_heads);
        c.small.owners = one_each + (c.tiles ? 0 : rows / few);
        c.small.waves = 8;
        c.small.merges = (long long)c.small.units * c.small.waves;
        c.small.parts = 2 * c.small.merges;
        c.small.entries = c.small.owners + c.small.parts;
    }
    if (c.tiles) {
        const long long longer = rows / (few + 1); /* requests that have tiles */
        c.tile.rows_per = TILE_SLOTS / group;
        c.tile.slots = (max_fresh < c.tile.rows_per ? max_fresh : c.tile.rows_per) * group;
        c.tile.units = units_of(blocks, kv_heads);
        c.tile.owners = rows / c.tile.rows_per + (longer < one_each ? longer : one_each);
        c.tile.waves = TILE_WAVES;
        c.tile.parts = (long long)c.tile.units * TILE_WAVES;
        c.tile.merges = c.tile.parts / 2;
        c.tile.entries = c.tile.owners > c.tile.parts ? c.tile.owners : c.tile.parts;
    }
    return c;
}
static __host__ __device__ __forceinline__ long long class_words(const Class &c) { return c.entries * ENTRY_WORDS + c.merges * MERGE_WORDS; }
static __host__ __device__ __forceinline__ long long schedule_words(const Caps &c) { return HEADER_WORDS + class_words(c.small) + class_words(c.tile); }
/* Offsets in a schedule, in words, and in a workspace, in floats. */
static __host__ __device__ __forceinline__ long long entries_at(const Caps &c, int tile) { return HEADER_WORDS + (tile ? class_words(c.small) : 0); }
static __host__ __device__ __forceinline__ long long merges_at(const Caps &c, int tile) {
    return entries_at(c, tile) + (tile ? c.tile.entries : c.small.entries) * ENTRY_WORDS;
}
static __host__ __device__ __forceinline__ long long parts_at(const Caps &c, int kv_heads, int tile) { return tile ? c.small.parts * kv_heads * c.small.slots * PART : 0; }
static __host__ __device__ __forceinline__ long long workspace_floats(const Caps &c, int kv_heads) {
    return parts_at(c, kv_heads, 1) + c.tile.parts * kv_heads * c.tile.slots * PART;
}
static __host__ __forceinline__ bool sizes_ok(int requests, long long rows, int max_fresh, int group, int kv_heads, int blocks) {
    return requests > 0 && requests <= NCB_PLAN_REQUESTS && rows >= 0 && rows <= (1ll << 26) && max_fresh > 0 && group > 0 && group <= MAX_GROUP &&
           kv_heads > 0 && kv_heads <= 65535 && blocks > 0 && blocks <= (1 << 20);
}

struct PagedArgs { /* of paged_attn's kernels */
    ncb_paged p;
    Caps caps;
    float scale_log2;
};

} /* namespace paged */
} /* namespace */
