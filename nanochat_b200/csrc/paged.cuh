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

constexpr int SPLIT_SLOTS = 64;   /* query slots of a block of the split kernel */
constexpr int MAX_GROUP = 64;     /* query heads per key/value head */
constexpr int MOST_WAVES = 4;     /* chunks are at least total / (MOST_WAVES * units): bounds entries, parts and merges */
constexpr int HEADER_WORDS = 16;  /* [0] entries, [1] merges */
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

/* Bounds of a schedule. An owner that is cut has more pages than a chunk, so all cut owners together are at most total / chunk, and their
 * chunks at most twice that. */
struct Caps {
    long long owners, entries, parts, merges;
    int slots; /* query slots of one part */
};
static __host__ __device__ __forceinline__ Caps caps_of(int requests, long long rows, int max_fresh, int group, int kv_heads, int blocks) {
    Caps c;
    const int rows_per = SPLIT_SLOTS / group, units = units_of(blocks, kv_heads);
    const long long one_each = requests < rows ? requests : rows;
    c.owners = one_each + rows / rows_per;
    c.parts = 2ll * units * MOST_WAVES;
    c.merges = (long long)units * MOST_WAVES;
    c.entries = c.owners + c.parts;
    c.slots = (max_fresh < rows_per ? max_fresh : rows_per) * group;
    return c;
}
static __host__ __device__ __forceinline__ long long schedule_words(const Caps &c) {
    return HEADER_WORDS + c.entries * ENTRY_WORDS + c.merges * MERGE_WORDS;
}
static __host__ __forceinline__ bool sizes_ok(int requests, long long rows, int max_fresh, int group, int kv_heads, int blocks) {
    return requests > 0 && requests <= NCB_PLAN_REQUESTS && rows >= 0 && rows <= (1ll << 26) && max_fresh > 0 && group > 0 && group <= MAX_GROUP &&
           kv_heads > 0 && kv_heads <= 65535 && blocks > 0 && blocks <= (1 << 20);
}

} /* namespace paged */
} /* namespace */
