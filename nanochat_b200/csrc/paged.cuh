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

constexpr int SPLIT_SLOTS = 64, TILE_SLOTS = 128; /* query slots of a block of the split kernel, of the tile kernel */
constexpr int MAX_GROUP = 64;                     /* query heads per key/value head */
constexpr int TILE_WAVES = 2;                     /* cut tiles are at most this often what runs at once */
constexpr int HEADER_WORDS = 16;                  /* entries and merges of the split kernel, of the tile kernel */
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

/* Bounds of a schedule, and where its parts lie. The tile kernel has the requests of more than SPLIT_SLOTS query slots, the split kernel the
 * others; where no request may have so many, no tile kernel runs, and the split kernel also has what is too long and only gets zeros.
 * A chunk of the split kernel is at least total / (waves * units) pages: the owners that are cut are at most waves * units, their
 * chunks at most twice that. Tiles are cut only where all entries are then at most TILE_WAVES * units. */
struct Class {
    long long owners, entries, merges, parts;
    int rows_per, slots; /* of an owner */
    int waves;
};
struct Caps {
    Class split, tile;
    int tiles; /* whether the tile kernel has anything */
};
static __host__ __device__ __forceinline__ Caps caps_of(int requests, long long rows, int max_fresh, int group, int kv_heads, int blocks) {
    Caps c = {};
    const int units = units_of(blocks, kv_heads);
    const long long one_each = requests < rows ? requests : rows;
    c.split.rows_per = SPLIT_SLOTS / group, c.tile.rows_per = TILE_SLOTS / group;
    c.tiles = max_fresh > c.split.rows_per;
    c.split.slots = (max_fresh < c.split.rows_per ? max_fresh : c.split.rows_per) * group;
    c.split.owners = one_each + (c.tiles ? 0 : rows / c.split.rows_per);
    c.split.waves = c.split.slots <= 16 ? 8 : 4;
    c.split.merges = (long long)units * c.split.waves;
    c.split.parts = 2 * c.split.merges;
    c.split.entries = c.split.owners + c.split.parts;
    if (c.tiles) {
        const long long longer = rows / (c.split.rows_per + 1); /* requests that have tiles */
        c.tile.slots = (max_fresh < c.tile.rows_per ? max_fresh : c.tile.rows_per) * group;
        c.tile.owners = rows / c.tile.rows_per + (longer < one_each ? longer : one_each);
        c.tile.waves = TILE_WAVES;
        c.tile.parts = (long long)units * TILE_WAVES;
        c.tile.merges = c.tile.parts / 2;
        c.tile.entries = c.tile.owners > c.tile.parts ? c.tile.owners : c.tile.parts;
    }
    return c;
}
static __host__ __device__ __forceinline__ long long class_words(const Class &c) { return c.entries * ENTRY_WORDS + c.merges * MERGE_WORDS; }
static __host__ __device__ __forceinline__ long long schedule_words(const Caps &c) { return HEADER_WORDS + class_words(c.split) + class_words(c.tile); }
/* Offsets in a schedule, in words, and in a workspace, in floats. */
static __host__ __device__ __forceinline__ long long entries_at(const Caps &c, int tile) { return HEADER_WORDS + (tile ? class_words(c.split) : 0); }
static __host__ __device__ __forceinline__ long long merges_at(const Caps &c, int tile) {
    return entries_at(c, tile) + (tile ? c.tile.entries : c.split.entries) * ENTRY_WORDS;
}
static __host__ __device__ __forceinline__ long long parts_at(const Caps &c, int kv_heads, int tile) { return tile ? c.split.parts * kv_heads * c.split.slots * PART : 0; }
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
