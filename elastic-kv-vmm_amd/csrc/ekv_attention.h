// What the attention kernels share: their arguments, and how the work of a launch is cut.
//
// A launch attends for sequences: a group's query tokens to its prefix, a batch row's to its own tokens or to both, or
// one query token's to its slots. A sequence has `rows` rows (query tokens x query heads of one KV head) in tiles of
// row_tile, and keys in units of unit; an item is one (sequence, KV head, row tile), and its key units are counted in one
// line over all items. Workgroup w takes places [w * quota, (w + 1) * quota) of that line, whatever the lengths are, so
// every workgroup has as many keys to read; but a cut inside an item of one or two units moves to the item's nearer end:
// starting and ending an item costs a workgroup about as much as reading a unit, so that cutting it would save nothing. An item cut between workgroups is joined by the merge kernel from the parts that
// each left (weighted values, largest score, sum). Places fit 31 bits: the host makes the unit larger where the tables'
// widths could pass them.
#pragma once

#include "../../include/ekv_kernels.h"
#include "ekv_common.h"
#include "ekv_fastdiv.h"
#include "ekv_tensor_util.h"
#include "ekv_wave.h"

#include <hip/hip_runtime.h>

#include <cmath>

namespace ekv {

// Token offset o of page p of KV head h: k + p * page_stride + o * token_stride + h * head_stride (bytes), V at
// + kv_stride.
struct Cache {
    const char* k;
    int64_t kv_stride;
    uint32_t page_stride, token_stride, head_stride;
    uint32_t pages, zero_below;   // ids zero_below .. pages - 1 name pages
    FastDiv page;                 // tokens per page
};

struct AttentionArgs {
    const char* query;
    int64_t q_token, q_head;      // bytes
    char* out;
    int64_t o_token, o_head;
    float* lse;
    int64_t l_token, l_head;      // elements
    Cache cache;
    const char* tables;           // [R, M] own pages of each request, or the slots of each query token
    int64_t table_row;            // bytes, as the columns' step
    const char* prefix_tables;    // [G, P]
    int64_t prefix_row;
    uint32_t table_col, prefix_col;
    int32_t requests;
    int32_t own_most, prefix_most;   // tokens that a table row covers
    IndexRef rows, lengths, query_starts, prefix_lengths, group_starts;
    int32_t table64, prefix64;
    int32_t tokens, batch, groups;
    int32_t heads, kv_heads, share, dim;   // share: query heads of a KV head
    FastDiv share_div;
    float scale;                  // of the scores, times log2 e; not negative
    uint32_t flip;                // the sign bits of two elements where the scale given was negative
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
    int32_t row_shift, unit_shift;   // row_tile and unit as powers of two
    int32_t workgroups;              // the most that take part
    int32_t direct;                  // an item that one workgroup has whole is written to the output
    int32_t dim_pad;
    int32_t slots;
    uint32_t alike_total;            // kSlots: places, and the items of a sequence and units of an item
    FastDiv alike_items, alike_units;
    float* parts;                    // slots of row_tile x dim_pad values, then row_tile largest scores and sums
    uint32_t* unit_starts;           // [sequences + 1] of the line, written for the merge
    uint32_t* item_starts;           // [sequences + 1]
};

// The arguments of a kernel. They are more words than a wave has scalar registers, and the compiler loads all of them
// first and spills what does not fit into vector registers; fresh() hides where they come from, so that each part of a
// kernel loads what it needs where it needs it.
struct Launch {
    AttentionArgs a;
    Phase p;
};

constexpr int kSeqChunk = 1024;      // sequences whose sums a workgroup holds at a time
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.0f;       // bits by which a weight may pass 1 before its row is scaled again

#if defined(__HIPCC__)

struct Sequence {
    int32_t first, count;       // query tokens
    int32_t prefix, own;        // keys of each kind
    int32_t newest;             // position of the last query token among the own tokens
    int32_t group, request;     // table rows (-1: none)
};

__device__ __forceinline__ const Launch& fresh() {
    auto at = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const Launch*)(at);
}

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
    return clamped(a.prefix_lengths.fetch(g), 0, a.prefix_most);
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
        q.own = a.own_most;
        q.newest = a.own_most;
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
        const int64_t length = a.lengths.fetch(s);
        const int64_t request = a.rows.data != nullptr ? a.rows.fetch(s) : s;
        q.request = request >= 0 && request < a.requests ? static_cast<int32_t>(request) : -1;
        q.own = q.request >= 0 ? clamped(length, 0, a.own_most) : 0;
        q.newest = clamped(length - 1, -1, 0x7ffffffe);
        q.group = mode == kWhole ? group_of(a, s) : -1;
        q.prefix = q.group >= 0 ? prefix_keys(a, q.group) : 0;
    }
    return q;
}

// Key units of a row tile: the prefix's, then the own tokens'. At least one, so that every row is somebody's work.
__device__ __forceinline__ int32_t prefix_units(const Sequence& q, const Phase& p) {
    return (q.prefix + (1 << p.unit_shift) - 1) >> p.unit_shift;
}

__device__ __forceinline__ int32_t units_of(const Sequence& q, const Phase& p) {
    return max(prefix_units(q, p) + ((q.own + (1 << p.unit_shift) - 1) >> p.unit_shift), 1);
}

__device__ __forceinline__ int32_t row_tiles_of(const AttentionArgs& a, const Sequence& q, const Phase& p) {
    return (q.count * a.share + (1 << p.row_shift) - 1) >> p.row_shift;
}

// Places of the line per workgroup.
__device__ __forceinline__ uint32_t quota_of(const Phase& p, uint32_t total) {
    return max((total + p.workgroups - 1) / p.workgroups, 1u);
}

// Whether an item keeps its cuts, and where the cut at place c goes that lies in the item of places
// [begin, begin + units). An item that moves its cuts has one at most.
__device__ __forceinline__ bool keeps_cuts(uint32_t units, uint32_t quota) { return units > min(quota, 2u); }

__device__ __forceinline__ uint32_t moved_cut(uint32_t c, uint32_t begin, uint32_t units, uint32_t quota) {
    return keeps_cuts(units, quota) ? c : (c - begin < begin + units - c ? begin : begin + units);
}

// How many own tokens a row of query token i (of the sequence's count) sees.
__device__ __forceinline__ int32_t seen_by(const Sequence& q, int32_t i) {
    return min(max(q.newest - q.count + i + 2, 0), q.own);
}

template <int kWaves>
struct LineCells {
    uint32_t units[kSeqChunk + 1];     // first place of each sequence of the chunk
    uint32_t items[kSeqChunk + 1];
    uint32_t sums[2][kWaves];
};

// The places and items of the sequences of one chunk, given what lies before it. All threads call it.
template <int kWaves>
__device__ __forceinline__ void line_chunk(const AttentionArgs& a, const Phase& p, int32_t chunk, uint32_t units_before,
                                           uint32_t items_before, LineCells<kWaves>& cells) {
    constexpr int kThreads = kWaves * 64;
    const int tid = threadIdx.x, wave = tid >> 6;
    const int32_t count = min(kSeqChunk, p.sequences - chunk);
    const int32_t per = (count + kThreads - 1) / kThreads;
    const int32_t first = min(tid * per, count), last = min(first + per, count);
    uint32_t units = 0, items = 0;
    __syncthreads();   // the cells' last use
#pragma unroll 1
    for (int32_t at = first; at < last; ++at) {
        const Sequence q = sequence_of(a, p.mode, chunk + at);
        const uint32_t mine = a.kv_heads * row_tiles_of(a, q, p);
        cells.units[at] = mine * units_of(q, p);
        cells.items[at] = mine;
        units += cells.units[at];
        items += mine;
    }
    const uint32_t unit_sum = wave_scan<kAdd>(units), item_sum = wave_scan<kAdd>(items);
    if ((tid & 63) == 63) {
        cells.sums[0][wave] = unit_sum, cells.sums[1][wave] = item_sum;
    }
    __syncthreads();
    uint32_t unit_at = units_before + unit_sum - units, item_at = items_before + item_sum - items;
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) {
        unit_at += w < wave ? cells.sums[0][w] : 0;
        item_at += w < wave ? cells.sums[1][w] : 0;
    }
    const bool publish = blockIdx.x == 0 && p.unit_starts != nullptr;
#pragma unroll 1
    for (int32_t at = first; at < last; ++at) {
        const uint32_t my_units = cells.units[at], my_items = cells.items[at];
        cells.units[at] = unit_at;
        cells.items[at] = item_at;
        if (publish) {
            p.unit_starts[chunk + at] = unit_at;
            p.item_starts[chunk + at] = item_at;
        }
        unit_at += my_units;
        item_at += my_items;
        if (at == count - 1) {
            cells.units[count] = unit_at;
            cells.items[count] = item_at;
            if (publish && chunk + count == p.sequences) {
                p.unit_starts[p.sequences] = unit_at;
                p.item_starts[p.sequences] = item_at;
            }
        }
    }
    __syncthreads();
}

// What a workgroup does next: key units [begin, end) of the `units` of one item.
struct Segment {
    Sequence q;
    int32_t head, row_begin, rows;      // KV head; first row of the tile; rows of the whole sequence
    int32_t begin, end, units;
    int32_t slot;
};

// The item at a place of the line.
struct Item {
    int32_t s;                          // sequence
    uint32_t local;                     // item within the sequence
    uint32_t before;                    // items before the sequence
    uint32_t begin, units;              // its places
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// Calls body(segment) for every segment of this workgroup, in order; all threads take part.
template <int kWaves, typename Body>
__device__ __forceinline__ void for_segments(LineCells<kWaves>& cells, Body&& body) {
    const AttentionArgs& a = fresh().a;
    const Phase& p = fresh().p;
    const uint32_t w = blockIdx.x;
    const bool alike = p.mode == kSlots;   // every sequence is as long: places are divided, not searched
    uint32_t total = 0;
    if (alike) {
        total = p.alike_total;
    } else {
        uint32_t items = 0;
        for (int32_t chunk = 0; chunk < p.sequences; chunk += kSeqChunk) {
            line_chunk(a, p, chunk, total, items, cells);
            const int32_t count = min(kSeqChunk, p.sequences - chunk);
            total = cells.units[count];
            items = cells.items[count];
        }
        total = uniform(total);
    }
    const uint32_t quota = quota_of(p, total);
    uint32_t at = w * quota;
    if (at >= total) {
        return;
    }
    int32_t chunk = 0, count = min(kSeqChunk, p.sequences);
    if (!alike && p.sequences > kSeqChunk) {
        line_chunk(a, p, 0, 0, 0, cells);
    }
    // The item at `place`, which does not go back from call to call.
    const auto item_at = [&](uint32_t place) {
        Item i;
        if (alike) {
            const uint32_t item = p.alike_units.div(place);
            i.units = p.alike_units.divisor;
            i.begin = item * i.units;
            i.s = p.alike_items.div(item);
            i.before = i.s * p.alike_items.divisor;
            i.local = item - i.before;
            return i;
        }
        while (cells.units[count] <= place) {
            const uint32_t units_before = cells.units[count], items_before = cells.items[count];
            chunk += kSeqChunk;
            count = min(kSeqChunk, p.sequences - chunk);
            line_chunk(a, p, chunk, units_before, items_before, cells);
        }
        int32_t low = 0, high = count;
        while (high - low > 1) {
            const int32_t mid = (low + high) >> 1;
            if (cells.units[mid] <= place) {
                low = mid;
            } else {
                high = mid;
            }
        }
        const uint32_t begin = uniform(cells.units[low]), all = uniform(cells.units[low + 1]) - begin;
        i.before = uniform(cells.items[low]);
        const uint32_t items = uniform(cells.items[low + 1]) - i.before;
        i.s = uniform(chunk + low);
        i.units = all, i.local = 0;
        if (items > 1) {
            i.units = all / items;
            i.local = (place - begin) / i.units;
        }
        i.begin = begin + i.local * i.units;
        return i;
    };
    Item i = item_at(at);
    at = moved_cut(at, i.begin, i.units, quota);
    uint32_t end = w * quota + quota;
    if (at == i.begin + i.units && at < min(end, total)) {
        i = item_at(at);
    }
    bool last = false;
#pragma unroll 1
    while (at < total) {
        // The workgroup's end: its cut, moved if it lies in this item.
        if (end < i.begin + i.units) {
            end = moved_cut(end, i.begin, i.units, quota);
            last = true;
        }
        const uint32_t stop = min(end, i.begin + i.units);
        if (at >= stop) {
            break;
        }
        Segment g;
        {
            const Launch& l = fresh();
            g.q = sequence_of(l.a, l.p.mode, i.s);
            g.units = i.units;
            g.head = i.local, g.row_begin = 0;
            const uint32_t row_tiles = row_tiles_of(l.a, g.q, l.p);
            if (row_tiles > 1) {
                g.head = i.local / row_tiles;
                g.row_begin = (i.local - g.head * row_tiles) << l.p.row_shift;
            }
            g.rows = g.q.count * l.a.share;
            g.begin = at - i.begin;
            g.end = stop - i.begin;
            g.slot = w + i.before + i.local;
        }
        body(g);
        at = stop;
        if (last || at >= total || at >= end) {
            break;
        }
        i = item_at(at);
    }
}

#endif

// attention_narrow.hip: row tiles of 16 * tiles16 rows, units of at least 2^narrow_unit_shift keys, and the workgroups
// that share a compute unit.
int narrow_unit_shift();
int narrow_groups(int tiles16, int32_t dim_pad);
void launch_narrow(const AttentionArgs& a, const Phase& p, int32_t dtype, int tiles16, void* stream);

// attention_wide.hip: row tiles of 128 (row_shift 7) or 256 rows, units of at least 64 keys.
void launch_wide(const AttentionArgs& a, const Phase& p, int32_t dtype, void* stream);

}  // namespace ekv
