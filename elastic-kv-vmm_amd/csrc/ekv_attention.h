// What the attention kernels share: their arguments, and how the work of a launch is cut.
//
// A launch attends for sequences: a group's query tokens to its prefix, a batch row's to its own tokens or to both, or
// one query token's to its slots. A sequence has `rows` rows (query tokens x query heads of one KV head) in tiles of
// row_tile, and keys in units of unit; an item is one (sequence, KV head, row tile), and its key units are counted in
// one line over all items. Workgroup w takes places [w * quota, (w + 1) * quota) of that line, whatever the lengths
// are, so every workgroup has as many keys to read. But where a run has two places or more, an item of one or two units
// is not cut, the workgroup in whose run it begins has it whole: starting and ending an item costs a workgroup about as
// much as reading a unit, so that cutting it would save nothing. An item cut between workgroups is joined from the parts
// that each left (weighted values, largest score, sum). Places fit 31 bits: the host makes the unit larger where the
// tables' widths could pass them.
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
    int32_t workgroups;              // that take part; of a launch of two phases, that both share
    int32_t weight;                  // cost of a unit, as the phases of a launch share its workgroups
    int32_t direct;                  // an item that one workgroup has whole is written to the output
    int32_t dim_pad;
    int32_t items;                   // at most, whatever the lengths are
    int32_t by_workgroup;            // how parts are numbered (part_slot)
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
    Phase p[2];        // own tokens (or all), prefixes
};

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.0f;       // bits by which a weight may pass 1 before its row is scaled again

#if defined(__HIPCC__)

// What a key that is not seen reads: weight 0 must meet a finite V.
__device__ __align__(256) static const uint32_t zero_row[128] = {};

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

// A lane's number, hidden likewise: what follows from it is computed where it is used, not once at the kernel's start
// and spilled until then.
__device__ __forceinline__ int hidden(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A load of memory that is not LDS. The compiler cannot tell for an address that a select chose, and its load for either
// kind returns in no order, so that a wait for one would wait for all that are under way.
template <typename V>
__device__ __forceinline__ V load_global(const char* at) {
    return *(const __attribute__((address_space(1))) V*)(at);
}

// A barrier for what is in LDS. __syncthreads() also waits for every load from memory that is under way, and would end
// each prefetch at the next barrier.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Keeps what stands beside it under its branch: without it the compiler computes a rare branch's selects every time.
__device__ __forceinline__ void rarely() { asm volatile(""); }

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
__device__ __forceinline__ uint32_t quota_of(uint32_t total, uint32_t workgroups) {
    return max((total + workgroups - 1) / workgroups, 1u);
}

// How many workgroups of a launch of two phases work on prefixes; the others work on own tokens. A prefix unit leaves as
// many bytes of parts as four hold of keys, so that a workgroup takes no fewer than two of them: with two, three, four
// and six 4 requests behind 1024 tokens take 20, 25, 22 and 28 us, 24 behind 5000 with drafts 35, 35, 35 and 36
// (bfloat16, head sizes 128 and 96). Beyond that the phases share the workgroups by their units' costs.
__device__ __forceinline__ uint32_t prefix_workgroups(const Phase& own, const Phase& prefix, uint32_t own_total,
                                                      uint32_t prefix_total) {
    const uint32_t all = own.workgroups, most = (prefix_total + 1) / 2;
    if (most + own_total <= all) {
        return most;
    }
    const int down = max(0, 15 - __builtin_clz(max(own_total, prefix_total) | 1));   // 17 bits of each are kept
    const uint32_t a = (prefix_total >> down) * prefix.weight, b = (own_total >> down) * own.weight;
    const uint32_t share = (all * a + (a + b) / 2) / max(a + b, 1u);
    return min(min(max(share, 1u), all - 1), most);
}

// Whether an item may be cut, and where the cut at place c goes that lies in the item of places [begin, begin + units):
// one that is not cut has at most one inside, and that moves to its end.
__device__ __forceinline__ bool keeps_cuts(uint32_t units, uint32_t quota) { return units > min(quota, 2u); }

__device__ __forceinline__ uint32_t moved_cut(uint32_t c, uint32_t begin, uint32_t units, uint32_t quota) {
    return c == begin || keeps_cuts(units, quota) ? c : begin + units;
}

// Where workgroup w leaves its part of an item that begins in the run of workgroup `first`, the `item`-th of the line.
// Where items that one workgroup has whole are written to the output, the items that leave parts begin in runs of their own
// and one ends before the next begins: first + w differs from part to part, and there are fewer than two a workgroup.
// Parts are numbered so where there are more items than workgroups, and else by item and workgroup.
__device__ __forceinline__ uint32_t part_slot(const Phase& p, uint32_t w, uint32_t first, uint32_t item) {
    return w + (p.by_workgroup != 0 ? first : item);
}

// How many own tokens a row of query token i (of the sequence's count) sees.
__device__ __forceinline__ int32_t seen_by(const Sequence& q, int32_t i) {
    return min(max(q.newest - q.count + i + 2, 0), q.own);
}

// A line's sequences, kChunk at a time.
template <int kWaves, int kChunk>
struct LineCells {
    uint32_t units[kChunk + 1];        // first place of each sequence of the chunk
    uint32_t items[kChunk + 1];
    uint32_t sums[2][kWaves];
    Sequence sequences[kChunk];
};

// The sequence that this thread has of a chunk, left in the cells, with its places and items.
struct Share {
    uint32_t units = 0, items = 0;
    uint32_t unit_sum = 0, item_sum = 0;   // inclusive over the wave
};

template <int kWaves, int kChunk>
__device__ __forceinline__ Share line_read(const AttentionArgs& a, const Phase& p, int32_t chunk,
                                           LineCells<kWaves, kChunk>& cells) {
    Share r;
    const int tid = threadIdx.x;
    if (tid < min(kChunk, p.sequences - chunk)) {
        const Sequence q = sequence_of(a, p.mode, chunk + tid);
        cells.sequences[tid] = q;
        r.items = a.kv_heads * row_tiles_of(a, q, p);
        r.units = r.items * units_of(q, p);
    }
    return r;
}

template <int kWaves, int kChunk>
__device__ __forceinline__ void line_scan(Share& r, LineCells<kWaves, kChunk>& cells) {
    r.unit_sum = wave_scan<kAdd>(r.units), r.item_sum = wave_scan<kAdd>(r.items);
    if ((threadIdx.x & 63) == 63) {
        cells.sums[0][threadIdx.x >> 6] = r.unit_sum, cells.sums[1][threadIdx.x >> 6] = r.item_sum;
    }
}

// After a barrier: the chunk's first places, given what lies before it.
template <int kWaves, int kChunk>
__device__ __forceinline__ void line_write(const Phase& p, int32_t chunk, const Share& r, uint32_t units_before,
                                           uint32_t items_before, LineCells<kWaves, kChunk>& cells) {
    const int tid = threadIdx.x, wave = tid >> 6;
    const int32_t count = min(kChunk, p.sequences - chunk);
    uint32_t unit_at = units_before + r.unit_sum - r.units, item_at = items_before + r.item_sum - r.items;
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) {
        unit_at += w < wave ? cells.sums[0][w] : 0;
        item_at += w < wave ? cells.sums[1][w] : 0;
    }
    // The thread after the last sequence's leaves the end (there is one: a chunk has fewer sequences than threads).
    static_assert(kChunk < kWaves * 64, "a thread past the chunk's last sequence");
    if (tid <= count) {
        cells.units[tid] = unit_at, cells.items[tid] = item_at;
        if (blockIdx.x == 0 && p.unit_starts != nullptr) {
            // The end is written over by the next chunk's first.
            p.unit_starts[chunk + tid] = unit_at, p.item_starts[chunk + tid] = item_at;
        }
    }
}

// The sequences of one chunk and their places. All threads call it.
template <int kWaves, int kChunk>
__device__ __forceinline__ void line_chunk(const AttentionArgs& a, const Phase& p, int32_t chunk, uint32_t units_before,
                                           uint32_t items_before, LineCells<kWaves, kChunk>& cells) {
    lds_barrier();   // the cells' last use
    Share r = line_read(a, p, chunk, cells);
    line_scan(r, cells);
    lds_barrier();
    line_write(p, chunk, r, units_before, items_before, cells);
    lds_barrier();
}

// What a workgroup does next: key units [begin, end) of the `units` of one item.
struct Segment {
    Sequence q;
    int32_t head, row_begin, rows;      // KV head; first row of the tile; rows of the whole sequence
    int32_t begin, end, units;
    int32_t slot;
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ Sequence uniform(const Sequence& q) {
    Sequence r;
    r.first = uniform(q.first), r.count = uniform(q.count);
    r.prefix = uniform(q.prefix), r.own = uniform(q.own), r.newest = uniform(q.newest);
    r.group = uniform(q.group), r.request = uniform(q.request);
    return r;
}

// The places of both phases' lines; the cells hold their first chunks where the lines have no more. All threads call it.
template <int kWaves, int kChunk>
__device__ __forceinline__ void line_totals(uint32_t (&totals)[2], LineCells<kWaves, kChunk> (&cells)[2]) {
    const Launch& l = fresh();
    uint32_t items[2] = {0, 0};
    totals[0] = totals[1] = 0;
    const int32_t longest = max(l.p[0].sequences, l.p[1].sequences);
#pragma unroll 1
    for (int32_t chunk = 0; chunk < longest; chunk += kChunk) {
        // Both lines' loads are under way together.
        lds_barrier();
        Share own = line_read(l.a, l.p[0], chunk, cells[0]), prefix = line_read(l.a, l.p[1], chunk, cells[1]);
        line_scan(own, cells[0]);
        line_scan(prefix, cells[1]);
        lds_barrier();
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            if (chunk < l.p[side].sequences) {
                line_write(l.p[side], chunk, side == 0 ? own : prefix, totals[side], items[side], cells[side]);
            }
        }
        lds_barrier();
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const int32_t count = min(kChunk, l.p[side].sequences - chunk);
            if (count > 0) {
                totals[side] = uniform(cells[side].units[count]), items[side] = uniform(cells[side].items[count]);
            }
        }
    }
}

// The place in the line's order of the b-th of `count` workgroups. Workgroups are dealt to the eight dies in turn: so each
// die gets a run of the line, and the heads of a request, which read neighbouring pieces of the same rows, meet behind
// one L2. For own tokens in pages of one, head size 64, 65 us instead of 69; at a page of 16 or 64, a head size of 128,
// for prefixes, prompts and Top-K slots it changed nothing or lost 1 us, so those go by the grid's order.
__device__ __forceinline__ uint32_t on_die(uint32_t b, uint32_t count) {
    const uint32_t die = b & 7, each = count >> 3, more = count & 7;
    return die * each + min(die, more) + (b >> 3);
}

// Calls body(segment) for every segment of phase `which` that workgroup w of those that share it has, in order; all
// threads take part. A phase whose sequences are one chunk may have its total and cells from line_totals.
//
// What runs once per workgroup or item costs as much as its instructions' way from memory, so this is kept short:
// sequences are read once and wait in LDS, and one copy of each step serves all cases.
template <int kWaves, int kChunk, typename Body>
__device__ __forceinline__ void for_segments(int which, uint32_t w, uint32_t workgroups, bool read, uint32_t total_read,
                                             LineCells<kWaves, kChunk>& cells, Body&& body) {
    const AttentionArgs& a = fresh().a;
    const Phase& p = fresh().p[which];
    const bool alike = p.mode == kSlots;   // every sequence is as long: places are divided, not searched
    const bool ready = alike || (read && p.sequences <= kChunk);
    uint32_t total = alike ? p.alike_total : total_read, quota = 0, at = 0, end = 0, units_before = 0, items_before = 0;
    int32_t chunk = 0;
    bool known = false, starting = true;
#pragma unroll 1
    while (true) {
        const int32_t count = min(kChunk, p.sequences - chunk);
        if (!ready) {
            line_chunk(a, p, chunk, units_before, items_before, cells);
            units_before = uniform(cells.units[count]), items_before = uniform(cells.items[count]);
        }
        if (!known) {
            if (!ready && chunk + kChunk < p.sequences) {
                chunk += kChunk;
                continue;
            }
            total = ready ? total : units_before;
            units_before = total;
            quota = quota_of(total, workgroups);
            at = w * quota, end = at + quota;
            known = true;
            if (at >= total) {
                return;
            }
            if (chunk > 0) {
                chunk = 0, units_before = 0, items_before = 0;
                continue;
            }
        }
#pragma unroll 1
        while (alike || at < units_before) {
            // The item at `at`: its sequence, which of the sequence's items it is, its places.
            uint32_t s, local = 0, before, begin, units;
            if (alike) {
                units = p.alike_units.divisor;
                const uint32_t item = p.alike_units.div(at);
                begin = item * units;
                s = p.alike_items.div(item);
                before = s * p.alike_items.divisor;
                local = item - before;
            } else {
                int32_t low = 0, high = count;
                while (high - low > 1) {
                    const int32_t mid = (low + high) >> 1;
                    const bool here = cells.units[mid] <= at;
                    low = here ? mid : low;
                    high = here ? high : mid;
                }
                s = uniform(low);
                begin = uniform(cells.units[s]);
                units = uniform(cells.units[s + 1]) - begin;
                if (at - begin >= units) {
                    return;     // only if the starts were not in order: places may have passed 32 bits
                }
                before = uniform(cells.items[s]);
                const uint32_t items = uniform(cells.items[s + 1]) - before;
                if (items > 1) {
                    units = units / items;
                    local = (at - begin) / units;
                    begin += local * units;
                }
            }
            if (starting) {
                starting = false;
                at = moved_cut(at, begin, units, quota);
                if (at == begin + units) {
                    if (at >= total) {
                        return;
                    }
                    continue;
                }
            }
            uint32_t stop = begin + units;
            const bool last = end < stop;
            stop = last ? moved_cut(end, begin, units, quota) : stop;
            if (at >= stop) {
                return;
            }
            Segment g;
            g.q = alike ? sequence_of(a, kSlots, s) : uniform(cells.sequences[s]);
            g.units = units;
            g.head = local, g.row_begin = 0;
            const uint32_t row_tiles = row_tiles_of(a, g.q, p);
            if (row_tiles > 1) {
                g.head = local / row_tiles;
                g.row_begin = (local - g.head * row_tiles) << p.row_shift;
            }
            g.rows = g.q.count * a.share;
            g.begin = at - begin;
            g.end = stop - begin;
            g.slot = part_slot(p, w, at == begin || p.by_workgroup == 0 ? w : begin / quota, before + local);
            body(g);
            at = stop;
            if (last || at >= end || at >= total) {
                return;
            }
        }
        chunk += kChunk;
    }
}

// Where a part holds four values, elements 4 quad .. 4 quad + 3 of row `row` of its tile, in 16-byte units: in the order
// of the registers that they come from, so that a wave's store is one run of memory.
__device__ __forceinline__ uint32_t narrow_place(int32_t row_shift, uint32_t row, uint32_t quad) {
    return ((((quad >> 2) << (row_shift - 4)) + (row >> 4)) << 6) + ((quad & 3) << 4) + (row & 15);
}

__device__ __forceinline__ uint32_t wide_place(int32_t dim_pad, uint32_t row, uint32_t quad) {
    return (((row >> 5) * (dim_pad >> 3) + (quad >> 1)) << 6) + ((quad & 1) << 5) + (row & 31);
}

#endif

// attention_narrow.hip: row tiles of 16 * tiles16 rows, units of at least 2^kNarrowUnit keys, and the workgroups that
// share a compute unit.
constexpr int kNarrowUnit = 7;
int narrow_groups(int tiles16, int32_t dim_pad);
void launch_narrow(const Launch& l, int32_t dtype, int tiles16, void* stream);

// attention_wide.hip: row tiles of 128 (row_shift 7) or 256 rows, units of at least 2^kWideUnit keys.
constexpr int kWideUnit = 6;
void launch_wide(const Launch& l, int32_t dtype, void* stream);

// attention_pair.hip: own tokens by the kernel for few rows (16) or for many (128), prefixes by the one for many.
void launch_pair(const Launch& l, int32_t dtype, void* stream);

}  // namespace ekv
