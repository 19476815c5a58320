// Layout of an adapter plan: a batch's tokens grouped by adapter, and the pieces of work that the
// low-rank adapter kernels take from it.  One int32 buffer; the tables come first so that their
// 16-byte entries are aligned.
#pragma once
#include "common.hpp"

namespace mi {
namespace adapters {

constexpr uint32_t kTile = 64;        // tokens of one adapter that a workgroup takes together
constexpr uint32_t kMaxChunk = 512;
constexpr uint32_t kMaxAdapters = 1024;
// A grid has at most 65535 workgroups along its second axis, where chunks are: 2^24 tokens and 1024 adapters give
// 33793.  Along the first are tiles times parts of K or N, below 2^32 threads; columns are counted in 32 bits.
constexpr uint64_t kMaxTokens = 1u << 24;
constexpr uint32_t kMaxWidth = 1u << 22;

struct Tile {  // positions [first, first + count) of the grouped order; adapter == n: tokens without one
    int32_t adapter, first, count, unused;
};
struct Chunk {  // slot: row of partial sums, or -1 where the adapter has no other chunk
    int32_t adapter, first, count, slot, tile, unused[3];
};

struct PlanLayout {
    uint32_t chunk;  // tokens of one adapter behind one partial weight gradient: few where there are few to share out
    uint64_t max_tiles, max_chunks, max_slots;
    uint64_t chunks, counts, slot_start, order, starts, histograms, size;  // offsets in int32; tiles are at 0
    uint32_t groups;  // workgroups that sort, each with a histogram, where one is too few; 0: one does everything

    __host__ __device__ PlanLayout(uint64_t tokens, uint32_t n)
    {
        const uint64_t used = tokens < n + 1ull ? tokens : n + 1ull;  // at most so many adapters
        max_tiles = tokens / kTile + used;
        chunk = tokens < 4096u ? 128u : tokens < 8192u ? 256u : 512u;
        max_chunks = tokens / chunk + used;
        // only adapters with more than `chunk` tokens have slots: at most n and at most tokens / chunk of them, each
        // with ceil(c / chunk) <= floor(c / chunk) + 1, and the floors add up to at most tokens / chunk
        max_slots = tokens / chunk + (n < tokens / chunk ? n : tokens / chunk);
        chunks = 4u * max_tiles;
        counts = chunks + 8u * max_chunks;  // {tiles, chunks}
        slot_start = counts + 2u;           // [n]
        order = slot_start + n;             // [tokens]
        starts = order + tokens;            // [n + 1]
        histograms = starts + n + 1u;
        groups = tokens <= 4096u ? 0u : tokens <= 256u * 1024u ? (uint32_t)((tokens + 1023u) / 1024u) : 256u;
        size = histograms + (uint64_t)groups * (n + 1u);
    }
};

}  // namespace adapters
}  // namespace mi
