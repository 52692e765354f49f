// What the attention kernels share: their arguments, and how the work of a launch is cut.
//
// A launch attends for sequences: a group's query tokens to its prefix, a batch row's to its own tokens or to both, or
// one query token's to its slots. A sequence has `rows` rows (query tokens x query heads of one KV head) in tiles of
// row_tile, and keys in tiles of key_tile; an item is one (sequence, KV head, row tile), and its key tiles are counted in
// one line over all items. Workgroup w of W takes places [w * total / W, (w + 1) * total / W) of that line, whatever the
// lengths are, so every workgroup has the same number of key tiles to read; an item cut between workgroups is joined by
// the merge kernel from the parts that each left (weighted values, largest score, sum).
#pragma once

#include "../../include/ekv_kernels.h"
#include "ekv_common.h"
#include "ekv_fastdiv.h"
#include "ekv_tensor_util.h"
#include "ekv_wave.h"

#include <hip/hip_runtime.h>

#include <cmath>

namespace ekv {

// Token offset o of page p of one KV head: k + p * page_stride + o * token_stride (bytes), V at + kv_stride.
struct Cache {
    const char* k;
    int64_t kv_stride;
    int64_t page_stride, token_stride, head_stride;
    int64_t pages;        // ids zero_below .. pages - 1 name pages
    int64_t zero_below;
    FastDiv page;         // tokens per page
};

struct AttentionArgs {
    const char* query;
    int64_t q_token, q_head;      // bytes
    char* out;
    int64_t o_token, o_head;
    float* lse;
    int64_t l_token, l_head;      // elements
    Cache cache;
    const void* tables;           // [R, M] own pages of each request, or the slots of each query token
    int64_t table_row, table_col;
    int64_t requests, columns;
    const void* prefix_tables;    // [G, P]
    int64_t prefix_row, prefix_col;
    int64_t prefix_columns;
    IndexRef rows, lengths, query_starts, prefix_lengths, group_starts;
    int32_t table64, prefix64;
    int32_t tokens, batch, groups;
    int32_t heads, kv_heads, share, dim;   // share: query heads of a KV head
    FastDiv share_div;
    float scale;                  // of the scores, times log2 e
};

enum PhaseMode : int32_t {
    kPrefixes,   // sequences are groups: all their query tokens against their prefix
    kOwn,        // sequences are batch rows against their own tokens
    kWhole,      // sequences are batch rows against prefix and own tokens
    kSlots,      // sequences are query tokens against their slots
};

// One launch's cut and where its parts go.
struct Phase {
    PhaseMode mode;
    int32_t sequences;
    int32_t row_tile, key_tile;
    int32_t workgroups;           // the most that take part
    int32_t direct;               // an item that one workgroup has whole is written to the output
    float* parts;                 // slots of row_tile x dim_pad values, then row_tile largest scores and sums
    int32_t dim_pad;
    int64_t slots;
    int64_t* tile_starts;         // [sequences + 1] of the line, written for the merge
    int32_t* item_starts;         // [sequences + 1]
};

constexpr int kAttentionThreads = 256;
constexpr int kAttentionWaves = kAttentionThreads / 64;
constexpr int kSeqPer = 4;
constexpr int kSeqChunk = kAttentionThreads * kSeqPer;   // sequences whose sums a workgroup holds at a time
constexpr int kFewestTiles = 4;                          // a workgroup takes no fewer key tiles: one a wave
constexpr float kLn2 = 0.6931471805599453f;

#if defined(__HIPCC__)

struct Sequence {
    int32_t first, count;       // query tokens
    int32_t prefix, own;        // keys of each kind
    int64_t length;             // own tokens as given (the last query token's position is length - 1)
    int32_t group, request;     // table rows (-1: none)
};

__device__ __forceinline__ int32_t clamped(int64_t v, int64_t low, int64_t high) {
    return static_cast<int32_t>(v < low ? low : (v > high ? high : v));
}

__device__ __forceinline__ int32_t first_token(const AttentionArgs& a, int32_t b) {
    return a.query_starts.data != nullptr ? clamped(a.query_starts.fetch(b), 0, a.tokens) : b;
}

__device__ __forceinline__ int32_t first_row(const AttentionArgs& a, int32_t g) {
    return a.group_starts.data != nullptr ? clamped(a.group_starts.fetch(g), 0, a.batch) : (g == 0 ? 0 : a.batch);
}

__device__ __forceinline__ int32_t prefix_keys(const AttentionArgs& a, int32_t g) {
    return clamped(a.prefix_lengths.fetch(g), 0, a.prefix_columns * a.cache.page.divisor);
}

// The group that batch row b belongs to, or -1: the last whose first row is not past b, if it reaches b.
__device__ __forceinline__ int32_t group_of(const AttentionArgs& a, int32_t b) {
    if (a.groups == 0) {
        return -1;
    }
    int32_t low = 0, high = a.groups;
    while (high - low > 1) {
        const int32_t mid = (low + high) >> 1;
        if (first_row(a, mid) <= b) {
            low = mid;
        } else {
            high = mid;
        }
    }
    return first_row(a, low) <= b && b < first_row(a, low + 1) ? low : -1;
}

__device__ __forceinline__ Sequence sequence_of(const AttentionArgs& a, PhaseMode mode, int32_t s) {
    Sequence q{};
    if (mode == kSlots) {
        q.first = s, q.count = 1;
        q.own = static_cast<int32_t>(a.columns);
        q.length = a.columns;
        q.group = -1, q.request = s;
    } else if (mode == kPrefixes) {
        const int32_t begin = first_row(a, s), end = first_row(a, s + 1);
        q.first = first_token(a, begin);
        q.count = max(first_token(a, max(begin, end)) - q.first, 0);
        q.prefix = prefix_keys(a, s);
        q.group = s, q.request = -1;
    } else {
        q.first = first_token(a, s);
        q.count = a.query_starts.data != nullptr ? max(first_token(a, s + 1) - q.first, 0) : 1;
        q.length = a.lengths.fetch(s);
        const int64_t request = a.rows.data != nullptr ? a.rows.fetch(s) : s;
        q.request = request >= 0 && request < a.requests ? static_cast<int32_t>(request) : -1;
        q.own = q.request >= 0 ? clamped(q.length, 0, a.columns * a.cache.page.divisor) : 0;
        q.group = mode == kWhole ? group_of(a, s) : -1;
        q.prefix = q.group >= 0 ? prefix_keys(a, q.group) : 0;
    }
    return q;
}

// Key tiles of a row tile: at least one, so that every row of a sequence is somebody's work.
__device__ __forceinline__ int32_t tiles_of(const Sequence& q, const Phase& p) {
    const int32_t k = p.key_tile;
    return max((q.prefix + k - 1) / k + (q.own + k - 1) / k, 1);
}

__device__ __forceinline__ int32_t row_tiles_of(const AttentionArgs& a, const Sequence& q, const Phase& p) {
    return (q.count * a.share + p.row_tile - 1) / p.row_tile;
}

// How many workgroups take part in a line of `total` key tiles, and the place where workgroup w begins.
__device__ __forceinline__ int32_t active_workgroups(const Phase& p, int64_t total) {
    return clamped(total / kFewestTiles, 1, p.workgroups);
}

__device__ __forceinline__ int64_t line_begin(int64_t total, int32_t w, int32_t active) {
    return total * w / active;
}

// The workgroup that has place t: the last w with total * w / active <= t.
__device__ __forceinline__ int32_t line_owner(int64_t total, int64_t t, int32_t active) {
    return static_cast<int32_t>(((t + 1) * active - 1) / total);
}

struct LineCells {
    int64_t tiles[kSeqChunk + 1];     // first place of each sequence of the chunk
    int32_t items[kSeqChunk + 1];
    uint32_t sums[3][kAttentionWaves];
};

// The places and items of the sequences of one chunk, given what lies before it. All threads call it.
__device__ __forceinline__ void line_chunk(const AttentionArgs& a, const Phase& p, int32_t chunk, int64_t tiles_before,
                                           int32_t items_before, LineCells& cells) {
    const int tid = threadIdx.x, wave = tid >> 6;
    const int32_t count = min(kSeqChunk, p.sequences - chunk);
    int64_t tiles = 0;
    uint32_t items = 0;
    __syncthreads();   // the cells' last use
#pragma unroll 1
    for (int k = 0; k < kSeqPer && tid * kSeqPer + k < count; ++k) {
        const int at = tid * kSeqPer + k;
        const Sequence q = sequence_of(a, p.mode, chunk + at);
        const int32_t mine = a.kv_heads * row_tiles_of(a, q, p);
        cells.tiles[at] = static_cast<int64_t>(mine) * tiles_of(q, p);
        cells.items[at] = mine;
        tiles += cells.tiles[at];
        items += mine;
    }
    // A thread's tiles stay below 2^40; 20 bits of them at a time keep the sums of 256 threads in 32 bits.
    const uint32_t low = static_cast<uint32_t>(tiles) & 0xfffffu;
    const uint32_t high = static_cast<uint32_t>(tiles >> 20);
    const uint32_t low_sum = wave_scan<kAdd>(low), high_sum = wave_scan<kAdd>(high), item_sum = wave_scan<kAdd>(items);
    if ((tid & 63) == 63) {
        cells.sums[0][wave] = low_sum, cells.sums[1][wave] = high_sum, cells.sums[2][wave] = item_sum;
    }
    __syncthreads();
    int64_t tile_at = tiles_before + static_cast<int64_t>(low_sum - low) + (static_cast<int64_t>(high_sum - high) << 20);
    int32_t item_at = items_before + static_cast<int32_t>(item_sum - items);
#pragma unroll
    for (int w = 0; w < kAttentionWaves - 1; ++w) {
        if (w < wave) {
            tile_at += static_cast<int64_t>(cells.sums[0][w]) + (static_cast<int64_t>(cells.sums[1][w]) << 20);
            item_at += static_cast<int32_t>(cells.sums[2][w]);
        }
    }
    const bool publish = blockIdx.x == 0 && p.tile_starts != nullptr;
#pragma unroll 1
    for (int k = 0; k < kSeqPer && tid * kSeqPer + k < count; ++k) {
        const int at = tid * kSeqPer + k;
        const int64_t mine = cells.tiles[at];
        const int32_t my_items = cells.items[at];
        cells.tiles[at] = tile_at;
        cells.items[at] = item_at;
        if (publish) {
            p.tile_starts[chunk + at] = tile_at;
            p.item_starts[chunk + at] = item_at;
        }
        tile_at += mine;
        item_at += my_items;
        if (at == count - 1) {
            cells.tiles[count] = tile_at;
            cells.items[count] = item_at;
            if (publish && chunk + count == p.sequences) {
                p.tile_starts[p.sequences] = tile_at;
                p.item_starts[p.sequences] = item_at;
            }
        }
    }
    __syncthreads();
}

// What a workgroup does next: key tiles [begin, end) of one item.
struct Segment {
    Sequence q;
    int32_t head, row_begin, rows;      // KV head; first row of the tile; rows of the whole sequence
    int32_t begin, end, tiles;
    int32_t slot;
};

// Calls body(segment) for every segment of this workgroup, in order; all threads take part.
template <typename Body>
__device__ __forceinline__ void for_segments(const AttentionArgs& a, const Phase& p, LineCells& cells, Body&& body) {
    const int32_t w = blockIdx.x;
    const bool alike = p.mode == kSlots;   // every sequence is as long: places are divided, not searched
    int64_t total = 0;
    int32_t alike_items = 0, alike_tiles = 1;
    if (alike) {
        const Sequence any = sequence_of(a, kSlots, 0);
        alike_tiles = tiles_of(any, p);
        alike_items = a.kv_heads * row_tiles_of(a, any, p);
        total = static_cast<int64_t>(p.sequences) * alike_items * alike_tiles;
    } else {
        int32_t items = 0;
        for (int32_t chunk = 0; chunk < p.sequences; chunk += kSeqChunk) {
            line_chunk(a, p, chunk, total, items, cells);
            const int32_t count = min(kSeqChunk, p.sequences - chunk);
            total = cells.tiles[count];
            items = cells.items[count];
        }
    }
    const int32_t active = active_workgroups(p, total);
    if (total == 0 || w >= active) {
        return;
    }
    int64_t at = line_begin(total, w, active);
    const int64_t end = line_begin(total, w + 1, active);
    int32_t chunk = 0, count = min(kSeqChunk, p.sequences);
    if (!alike && p.sequences > kSeqChunk) {
        line_chunk(a, p, 0, 0, 0, cells);
    }
    while (at < end) {
        int32_t s, item, before = 0;      // sequence, item within it, items before it
        int64_t local;
        if (alike) {
            const int64_t place = at / alike_tiles;
            s = static_cast<int32_t>(place / alike_items);
            item = static_cast<int32_t>(place % alike_items);
            before = s * alike_items;
            local = at - place * alike_tiles;
        } else {
            while (cells.tiles[count] <= at) {
                const int64_t tiles_before = cells.tiles[count];
                const int32_t items_before = cells.items[count];
                chunk += kSeqChunk;
                count = min(kSeqChunk, p.sequences - chunk);
                line_chunk(a, p, chunk, tiles_before, items_before, cells);
            }
            int32_t low = 0, high = count;
            while (high - low > 1) {
                const int32_t mid = (low + high) >> 1;
                if (cells.tiles[mid] <= at) {
                    low = mid;
                } else {
                    high = mid;
                }
            }
            low = __builtin_amdgcn_readfirstlane(low);
            s = chunk + low;
            before = cells.items[low];
            local = at - cells.tiles[low];
            item = 0;
        }
        Segment g;
        g.q = sequence_of(a, p.mode, s);
        g.tiles = tiles_of(g.q, p);
        if (!alike) {
            item = static_cast<int32_t>(local / g.tiles);
            local -= static_cast<int64_t>(item) * g.tiles;
        }
        const int32_t row_tiles = row_tiles_of(a, g.q, p);
        g.head = item / row_tiles;
        g.row_begin = item % row_tiles * p.row_tile;
        g.rows = g.q.count * a.share;
        g.begin = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(local));
        g.end = static_cast<int32_t>(min(static_cast<int64_t>(g.tiles), g.begin + (end - at)));
        g.slot = w + before + item;
        body(g);
        at += g.end - g.begin;
    }
}

#endif

// The launches of attention_narrow.hip and attention.hip's merge; the row tiles are 16 * tiles16.
void launch_narrow(const AttentionArgs& a, const Phase& p, int32_t dtype, int tiles16, void* stream);

}  // namespace ekv
