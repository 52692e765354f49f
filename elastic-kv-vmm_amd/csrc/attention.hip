// Attention of queries to the paged K/V pool (gfx950): behind a prefix that a group of requests shares, and over the
// Top-K slots of a decode step.
//
//   o = sum_j softmax_j(scale q . k_j) v_j,   lse = log sum_j exp(scale q . k_j)
//
// over the keys that a query token sees. With the running largest score m, the sum l = sum exp(s_j - m) and the
// weighted values a = sum exp(s_j - m) v_j, two parts of the keys join as m = max(m1, m2),
// l = l1 e^(m1 - m) + l2 e^(m2 - m), a likewise, and o = a / l; statistics and sums are held in 32 bits.
//
// The kernels that read K and V are in attention_narrow.hip, attention_wide.hip and attention_pair.hip; here are the
// checks, the choice of a launch, and the merge of the parts that a launch's workgroups leave of one item
// (ekv_attention.h).
#include "ekv_attention.h"
#include "ekv_mfma.h"
#include "ekv_pool.h"

#include <algorithm>
#include <limits>

namespace ekv {
namespace {

constexpr int kMergeThreads = 256, kMergeColumns = 8;
constexpr int kMergeByToken = 8;        // workgroups per compute unit up to which the merge goes by tokens

// The workgroups that hold a token's parts of one phase, and where.
struct Parts {
    const float* base;          // first part
    const float* stats;         // first part's largest score of the row; its sum is row_tile later
    int32_t step;               // to the next part
    int32_t row_tile;
    int32_t count;              // -1: the output is written already
    uint32_t inside;            // the row's place in its tile
    int32_t wide, dim_pad, row_shift;

    __device__ __forceinline__ uint32_t place(uint32_t quad) const {
        return (wide ? wide_place(dim_pad, inside, quad) : narrow_place(row_shift, inside, quad)) * 4;
    }
};

// The parts of row `row` (of one KV head) of sequence s: none when the sequence was nobody's work.
__device__ __forceinline__ Parts parts_of(const AttentionArgs& a, const Phase& p, uint32_t workgroups, int32_t s,
                                          int32_t head, int32_t row) {
    uint32_t begin, total, item, units, row_tiles;
    if (p.mode == kSlots) {
        units = p.alike_units.divisor;
        item = s * p.alike_items.divisor;
        row_tiles = row_tiles_of(a, sequence_of(a, kSlots, 0), p);
        begin = item * units;
        total = p.alike_total;
    } else {
        begin = p.unit_starts[s];
        item = p.item_starts[s];
        total = p.unit_starts[p.sequences];
        const uint32_t items = p.item_starts[s + 1] - item;
        if (items == 0) {
            return Parts{};
        }
        units = (p.unit_starts[s + 1] - begin) / items;
        row_tiles = items / a.kv_heads;
    }
    const uint32_t local = head * row_tiles + (row >> p.row_shift);
    begin += local * units;
    // Who has it: everyone with a place of it, or the one with its first place where it is not cut.
    const uint32_t quota = quota_of(total, workgroups), first = begin / quota;
    const uint32_t count = keeps_cuts(units, quota) ? (begin + units - 1) / quota - first + 1 : 1;
    Parts r;
    r.row_tile = 1 << p.row_shift;
    r.step = r.row_tile * (p.dim_pad + 2);
    const uint32_t slot = part_slot(p, first, first, item + local), inside = row & (r.row_tile - 1);
    const float* part = p.parts + static_cast<int64_t>(slot) * r.step;
    r.base = part;
    r.inside = inside;
    r.wide = p.row_shift > 6;
    r.dim_pad = p.dim_pad, r.row_shift = p.row_shift;
    r.stats = part + r.row_tile * p.dim_pad + inside;
    r.count = static_cast<int32_t>(count);
    if (p.direct != 0 && count == 1) {
        r.count = -1;
    } else if (count > static_cast<uint32_t>(p.slots) || slot > static_cast<uint32_t>(p.slots) - count) {
        r.count = 0;            // only if the starts were not in order
    }
    return r;
}

// Four elements of a row, joined over some of its parts.
struct Joined {
    float top = -INFINITY, sum = 0;
    f32x4 value = {0, 0, 0, 0};

    // Parts split, split + splits, ... of `count`, the own ones first and then the prefix's, the loads of kBatch parts in
    // flight.
    template <int kBatch>
    __device__ __forceinline__ void join(const Parts& mine, const Parts& theirs, int32_t own_count, int32_t count,
                                         uint32_t quad, int32_t split, int32_t splits) {
        const uint32_t my_place = mine.place(quad), their_place = theirs.place(quad);
        for (int32_t i = split; i < count; i += splits * kBatch) {
            float part_top[kBatch], part_sum[kBatch];
            f32x4 part_value[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int32_t at = i + k * splits;
                const bool there = at < count;
                const bool first = at < own_count;
                const int64_t place = there ? (first ? at : at - own_count) : 0;
                const bool from_own = there ? first : own_count > 0;
                const float* stats = (from_own ? mine.stats : theirs.stats) + place * (from_own ? mine.step : theirs.step);
                const float* base = (from_own ? mine.base : theirs.base) + place * (from_own ? mine.step : theirs.step);
                part_top[k] = stats[0];
                part_sum[k] = stats[from_own ? mine.row_tile : theirs.row_tile];
                part_value[k] = *reinterpret_cast<const f32x4*>(base + (from_own ? my_place : their_place));
                part_top[k] = there ? part_top[k] : -INFINITY;
            }
            float most = top;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                most = fmaxf(most, part_top[k]);
            }
            const float safe = rescale(most);
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                // A part that saw nothing holds zeros, or NaN where its scores were; only one that is not there is left out.
                const float factor = exp2f(part_top[k] - safe);
                const bool there = i + k * splits < count;
                sum += there ? part_sum[k] * factor : 0.0f;
                value += there ? part_value[k] * factor : f32x4{0, 0, 0, 0};
            }
        }
    }

    // Makes `most` the score that the sums are relative to; the score to subtract (0 where no key was seen).
    __device__ __forceinline__ float rescale(float most) {
        const float safe = most == -INFINITY ? 0.0f : most;
        const float keep = exp2f(top - safe);
        sum *= keep;
        value *= keep;
        top = most;
        return safe;
    }

    template <typename T>
    __device__ __forceinline__ void write(const AttentionArgs& a, int32_t token, int32_t row_head, int32_t quad) const {
        const float inverse = sum == 0 ? 0.0f : 1.0f / sum;
        *reinterpret_cast<words2*>(a.out + token * a.o_token + row_head * a.o_head + quad * 8) =
            words2{T::pack(value[0] * inverse, value[1] * inverse), T::pack(value[2] * inverse, value[3] * inverse)};
        if (quad == 0 && a.lse != nullptr) {
            a.lse[token * a.l_token + row_head * a.l_head] =
                sum == 0 ? -INFINITY : (top - T::kShift + log2f(sum)) * kLn2;
        }
    }
};

// One workgroup per (query token, KV head) and 256 pieces of four elements of its rows, for launches whose every row has
// parts and for those of few tokens. What bounds it is the latency of its loads (a row has as many parts as workgroups
// shared its keys), so a small row's parts are spread over the threads that it leaves idle, and joined through LDS, and
// a large share's pieces over workgroups: with one for all of 256 query heads a call took 114 us instead of 46.
// Measured: 4.4 us behind a Top-K step of 4 tokens, 10.8 us behind 32 tokens of 32 heads with 8192 keys of prefix (22 MB
// of parts).
template <typename T>
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(const AttentionArgs a, const Phase own,
                                                                  const Phase prefix) {
    __shared__ f32x4 s_value[kMergeThreads];
    __shared__ float s_top[kMergeThreads], s_sum[kMergeThreads];
    const int32_t token = blockIdx.x, head = blockIdx.y;
    int32_t b = token;
    if (own.mode != kSlots && a.query_starts.data != nullptr) {
        int32_t low = 0, high = a.batch;
        while (high - low > 1) {
            const int32_t mid = (low + high) >> 1;
            if (first_token(a, mid) <= token) {
                low = mid;
            } else {
                high = mid;
            }
        }
        b = a.batch > 0 && first_token(a, low) <= token && token < first_token(a, low + 1) ? low : -1;
    }
    const int32_t group = b >= 0 && prefix.sequences > 0 ? group_of(a, b) : -1;
    const int32_t own_first = b >= 0 && own.mode != kSlots ? first_token(a, b) : token;
    const int32_t prefix_first = group >= 0 ? first_token(a, first_row(a, group)) : 0;
    uint32_t own_workgroups = own.workgroups, shared = 0;
    if (prefix.sequences > 0) {
        shared = prefix_workgroups(own, prefix, own.unit_starts[own.sequences], prefix.unit_starts[prefix.sequences]);
        own_workgroups -= shared;
    }
    const int32_t quads = (a.dim + 3) >> 2, units = a.share * quads;
    const int32_t splits = units < kMergeThreads ? kMergeThreads / units : 1;
    for (int32_t begin = blockIdx.z * kMergeThreads; begin < units; begin += gridDim.z * kMergeThreads) {
        const int32_t split = splits > 1 ? threadIdx.x / units : 0;
        const int32_t unit = begin + threadIdx.x - split * units;
        const bool live = unit < units && split < splits;
        // Rows first: their values lie side by side.
        const int32_t quad = live ? a.share_div.div(unit) : 0, sub = live ? unit - quad * a.share : 0;
        Parts mine{}, theirs{};
        if (b >= 0) {
            mine = parts_of(a, own, own_workgroups, b, head, (token - own_first) * a.share + sub);
        }
        if (group >= 0) {
            theirs = parts_of(a, prefix, shared, group, head, (token - prefix_first) * a.share + sub);
        }
        const bool written = mine.count < 0;
        const int32_t own_count = max(mine.count, 0), count = live && !written ? own_count + theirs.count : 0;
        Joined joined;
        joined.template join<8>(mine, theirs, own_count, count, quad, split, splits);
        if (splits > 1) {
            s_top[threadIdx.x] = joined.top, s_sum[threadIdx.x] = joined.sum, s_value[threadIdx.x] = joined.value;
            __syncthreads();
            if (split == 0) {
                float most = joined.top;
                for (int32_t k = 1; k < splits; ++k) {
                    most = fmaxf(most, s_top[threadIdx.x + k * units]);
                }
                const float safe = joined.rescale(most);
                for (int32_t k = 1; k < splits; ++k) {
                    const float factor = exp2f(s_top[threadIdx.x + k * units] - safe);
                    joined.sum += s_sum[threadIdx.x + k * units] * factor;
                    joined.value += s_value[threadIdx.x + k * units] * factor;
                }
            }
        }
        if (live && !written && split == 0) {
            joined.write<T>(a, token, head * a.share + sub, quad);
        }
    }
}

// The cuts of a launch of one phase: the column of workgroups w joins the item that workgroup w begins and others go on
// with, if there is one; all other items are written already. The rows of tokens that belong to no batch row are zeroed
// here. What bounds it: the parts of 256 cut items of 256 rows, 68 MB in 22 us at a head size of 128.
template <typename T>
__global__ __launch_bounds__(kMergeThreads) void cuts_kernel(const AttentionArgs a, const Phase p) {
    const uint32_t total = p.mode == kSlots ? p.alike_total : p.unit_starts[p.sequences];
    const uint32_t quota = quota_of(total, p.workgroups), cut = (blockIdx.x + 1) * quota;
    const int32_t columns = gridDim.y * kMergeThreads, column = blockIdx.y * kMergeThreads + threadIdx.x;
    if (p.mode != kSlots && a.query_starts.data != nullptr) {
        // The batch rows' tokens lie side by side: the others are in front of them and behind.
        const int32_t front = a.batch > 0 ? first_token(a, 0) : 0, behind = a.batch > 0 ? first_token(a, a.batch) : 0;
        const int32_t gap = front + a.tokens - behind, quads = a.dim >> 2;
        for (int32_t i = blockIdx.x; i < gap; i += gridDim.x) {
            const int32_t token = i < front ? i : behind + i - front;
            for (int32_t unit = column; unit < a.heads * quads; unit += columns) {
                const int32_t head = unit / quads;
                Joined{}.write<T>(a, token, head, unit - head * quads);
            }
        }
    }
    if (cut >= total) {
        return;
    }
    int32_t s;
    uint32_t begin, units, items, local;
    if (p.mode == kSlots) {
        const uint32_t item = p.alike_units.div(cut);
        s = p.alike_items.div(item);
        items = p.alike_items.divisor, units = p.alike_units.divisor;
        begin = item * units, local = item - s * items;
    } else {
        int32_t low = 0, high = p.sequences;
        while (high - low > 1) {
            const int32_t mid = (low + high) >> 1;
            if (p.unit_starts[mid] <= cut) {
                low = mid;
            } else {
                high = mid;
            }
        }
        s = low;
        items = p.item_starts[s + 1] - p.item_starts[s];
        begin = p.unit_starts[s];
        units = p.unit_starts[s + 1] - begin;
        if (items == 0 || cut - begin >= units) {
            return;             // the latter only if the starts were not in order
        }
        units = max(units / items, 1u);
        local = (cut - begin) / units;
        begin += local * units;
    }
    if (begin == cut || begin < cut - quota || !keeps_cuts(units, quota)) {
        return;
    }
    const Sequence q = sequence_of(a, p.mode, s);
    const int32_t row_tiles = max(items / a.kv_heads, 1u), head = local / row_tiles;
    const int32_t row_begin = (local - head * row_tiles) << p.row_shift, rows = q.count * a.share - row_begin;
    Parts parts = parts_of(a, p, p.workgroups, s, head, row_begin);
    const float* stats = parts.stats;
    const int32_t quads = a.dim >> 2, count = parts.count;
    if (count < 1) {
        return;
    }
    for (int32_t unit = column; unit < quads << p.row_shift; unit += columns) {
        // Four rows of all quads: a wave reads pieces of 64 bytes and writes pieces of a row.
        const int32_t four = (unit >> 2) / quads, quad = (unit >> 2) - four * quads, row = four * 4 + (unit & 3);
        if (row >= rows) {
            continue;
        }
        parts.inside = row, parts.stats = stats + row;
        Joined joined;
        if (count <= 2) {
            joined.join<2>(parts, parts, count, count, quad, 0, 1);
        } else {
            joined.join<8>(parts, parts, count, count, quad, 0, 1);
        }
        const int32_t at = row_begin + row, token = a.share_div.div(at);
        joined.write<T>(a, q.first + token, head * a.share + at - token * a.share, quad);
    }
}

// ---------------------------------------------------------------- host

constexpr int64_t kMostHeads = 65535, kMostTokens = 1 << 23, kMostRows = int64_t{1} << 30,
                  kMostBatch = 1 << 20;
constexpr int32_t kComputeUnits = 256;

// Query, output, statistics and cache: what both entry points share.
AttentionArgs common_args(const ekv_tensor* query_p, const ekv_planes* planes, int64_t layer, int64_t kv_heads,
                 int64_t page_size, double scale, const ekv_tensor* out_p, const ekv_tensor* lse_p) {
    const ekv_tensor& query = need_rows(query_p, "query");
    const ekv_tensor& out = need_rows(out_p, "output");
    for (int d = 0; d < 3; ++d) {
        need_dim(out, d, query.shape[d], "output");
    }
    if (out.dtype != query.dtype) {
        throw std::invalid_argument("output must have the query's type");
    }
    AttentionArgs a{};
    const int64_t tokens = query.shape[0], heads = query.shape[1], dim = query.shape[2];
    if (kv_heads < 1 || heads < 1 || heads % kv_heads != 0) {
        throw std::invalid_argument("kv_heads must divide the query's heads");
    }
    if (dim < 8 || dim > 256 || dim % 8 != 0) {
        throw std::invalid_argument("the head size must be a multiple of 8 from 8 to 256");
    }
    if (heads > kMostHeads || tokens > kMostTokens || tokens > kMostRows / heads) {
        throw std::invalid_argument("more than 65535 heads, 2^23 query tokens or 2^30 query rows");
    }
    a.tokens = static_cast<int32_t>(tokens), a.heads = static_cast<int32_t>(heads), a.dim = static_cast<int32_t>(dim);
    a.kv_heads = static_cast<int32_t>(kv_heads);
    a.share = a.heads / a.kv_heads;
    a.share_div = FastDiv(static_cast<uint32_t>(a.share));
    const PlanePages pages = plane_pages(planes, layer, kv_heads * a.dim * 2, page_size, 2);
    Cache& c = a.cache;
    c.token_stride = static_cast<uint32_t>(pages.token_stride);
    c.page_stride = static_cast<uint32_t>(pages.page_stride);
    c.pages = static_cast<uint32_t>(pages.pages);
    c.head_stride = static_cast<uint32_t>(dim * 2);
    c.page = FastDiv(static_cast<uint32_t>(page_size));
    c.zero_below = 1;
    c.k = pages.at;
    c.kv_stride = pages.kv_stride;
    a.query = static_cast<const char*>(query.data);
    a.q_token = query.stride[0] * 2, a.q_head = query.stride[1] * 2;
    a.out = static_cast<char*>(out.data);
    a.o_token = out.stride[0] * 2, a.o_head = out.stride[1] * 2;
    if (lse_p != nullptr) {
        const ekv_tensor& lse = need(lse_p, "lse");
        need_ndim(lse, 2, "lse");
        need_dim(lse, 0, a.tokens, "lse");
        need_dim(lse, 1, a.heads, "lse");
        need_data(lse, "lse");
        if (lse.dtype != EKV_FLOAT32) {
            throw std::invalid_argument("lse must be float32");
        }
        a.lse = static_cast<float*>(lse.data);
        a.l_token = lse.stride[0], a.l_head = lse.stride[1];
    }
    // Log2 e: the kernels' exponentials have base two. A negative scale changes the queries' signs; zero is taken as the
    // smallest number, since an unseen key's score is minus infinity, which zero would make NaN.
    a.scale = static_cast<float>(std::fabs(scale) * 1.4426950408889634);
    if (!std::isfinite(a.scale)) {
        throw std::invalid_argument("scale must be finite");
    }
    a.scale = std::max(a.scale, std::numeric_limits<float>::min());
    a.flip = scale < 0 ? 0x80008000u : 0;
    return a;
}

uint64_t aligned(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

// The launch of a call and the workspace it uses.
struct Plan {
    int tiles16 = 0;           // 16-row tiles of the own tokens' kernel
    bool pair = false;         // own tokens and prefixes as two phases of one launch
    Phase own{}, prefix{};
    uint64_t bytes = 0;
};

int32_t padded_dim(int64_t dim) { return dim <= 64 ? 64 : (dim <= 96 ? 96 : (dim <= 128 ? 128 : 256)); }

// 16-row tiles that hold `rows` rows: 1, 2 or 4 of the kernel for few rows, 8 or 16 of the one for many (2 and 8 at most
// at 256 columns, where the registers hold no more). A tile that rows fill in part costs its whole products, several tiles
// read the keys several times. Calls of 32 requests of 2000 tokens, head size 128, us with tiles of 1, 2, 4, 8, 16:
//   16 rows, 8 KV heads   55  55  57  62  75        64 rows, 2 KV heads    53  36  31  36  34
//   32 rows, 8 KV heads   96  58  59  65  76       128 rows, 2 KV heads    92  54  42  41  38
//                                                  256 rows, 2 KV heads   173  99  60  53  46
// and at a head size of 256 with 1, 2, 8: 106 152 176 for 16 rows, 200 156 181 for 32, 94 83 71 for 64.
int tiles_for(int64_t rows, int32_t dim_pad) {
    if (rows <= 32) {
        return rows <= 16 ? 1 : 2;
    }
    if (rows <= 64 && dim_pad <= 128) {
        return 4;
    }
    return rows <= 128 || dim_pad > 128 ? 8 : 16;
}

// A phase's cut and its place in the workspace.
void cut(Plan& plan, Phase& p, PhaseMode mode, int64_t sequences, int tiles16, int64_t tokens, int64_t share,
         int64_t kv_heads, int32_t dim_pad, bool direct) {
    p.mode = mode;
    p.sequences = static_cast<int32_t>(sequences);
    p.row_shift = 4;
    while ((1 << p.row_shift) < 16 * tiles16) {
        ++p.row_shift;
    }
    p.unit_shift = tiles16 < 8 ? kNarrowUnit : kWideUnit;
    p.dim_pad = dim_pad;
    p.workgroups = kComputeUnits * (tiles16 < 8 ? narrow_groups(tiles16, dim_pad) : (tiles16 == 8 && dim_pad <= 128 ? 2 : 1));
    // A unit of the kernel for few rows is 128 keys read at the card's rate, one of the kernel for many 64 keys'
    // products. Weights of 3, 4, 5, 6 and 8 against 3 took 47, 46, 43, 41 and 46 us for 32 requests behind 8192 tokens,
    // 126, 122, 110, 124 and 130 for 128 requests behind 32768, 73, 68, 69, 69 and 69 for seven groups of 13: head sizes
    // 128, 128 and 64, 4, 8 and 4 query heads a KV head, pages of 16, 64 and 1. Other ratios of a unit's bytes to its
    // products rest on these three.
    p.weight = tiles16 < 8 ? 5 : 3;
    p.direct = direct;
    // Row tiles of all sequences: every sequence's last may be part-filled.
    const int64_t items = kv_heads * ((tokens * share >> p.row_shift) + std::min(sequences, tokens));
    if (items > (int64_t{1} << 30)) {
        throw std::invalid_argument("more than 2^30 row tiles");
    }
    p.items = static_cast<int32_t>(items);
    p.by_workgroup = direct && items > p.workgroups;
    p.slots = static_cast<int32_t>(p.workgroups + (p.by_workgroup ? p.workgroups : items));
    p.parts = reinterpret_cast<float*>(plan.bytes);
    plan.bytes += aligned((static_cast<uint64_t>(p.slots) << p.row_shift) * (dim_pad + 2) * sizeof(float));
    if (mode != kSlots) {
        p.unit_starts = reinterpret_cast<uint32_t*>(plan.bytes);
        plan.bytes += aligned((static_cast<uint64_t>(sequences) + 1) * sizeof(uint32_t));
        p.item_starts = reinterpret_cast<uint32_t*>(plan.bytes);
        plan.bytes += aligned((static_cast<uint64_t>(sequences) + 1) * sizeof(uint32_t));
    }
}

// Makes the unit so large that the line's places fit 31 bits, whatever the lengths on the device are.
void fit_units(Phase& p, int64_t keys) {
    while (p.items > 0 && (keys >> p.unit_shift) + 2 > 0x7fffffff / p.items) {
        ++p.unit_shift;
    }
}

void need_sizes(int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim) {
    if (tokens < 0 || sequences < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || dim < 8 || dim > 256) {
        throw std::invalid_argument("attention sizes must be positive, kv_heads a divisor of the heads and the head "
                                    "size from 8 to 256");
    }
    if (heads > kMostHeads || tokens > kMostTokens || tokens > kMostRows / heads || sequences > kMostBatch) {
        throw std::invalid_argument("more than 65535 heads, 2^23 query tokens, 2^30 query rows or 2^20 batch rows");
    }
}

Plan prefix_plan(int64_t tokens, int64_t batch, int64_t groups, int64_t heads, int64_t kv_heads, int64_t dim,
                 int64_t max_query) {
    need_sizes(tokens, std::max(batch, groups), heads, kv_heads, dim);
    if (groups < 0 || max_query < 1) {
        throw std::invalid_argument("max_query must be positive");
    }
    Plan plan;
    const int64_t share = heads / kv_heads, row_rows = std::min(max_query, tokens) * share;
    const int32_t dim_pad = padded_dim(dim);
    // Rows of a group fill tiles that a batch row's alone leave part-empty: then the prefix is a phase of its own. Where a
    // batch row has 64 rows both ways are even: 32 requests of 500 tokens behind 8192, head size 128, 8 KV heads, by
    // rows of a batch row 8, 16, 32, 64, 96: as phases 43, 63, 103, 159, 226 us, as one 134, 138, 142, 166, 199. Own
    // tokens of 17 rows and more go to the kernel for many rows: in tiles of 16 they are read once per tile, 32 rows of
    // 4000 tokens 242 us against 164 (of 500 tokens 92 against 100; 16 rows of 4000 tokens 142 against 149).
    // These were batches of like rows. The rule goes by the longest row, so a prompt piece makes every decode row beside
    // it read the prefix by itself: 127 rows of one token and one of 1024 behind 32768 tokens, 8 query heads a KV head,
    // take 1327 us in one call and 108 + 322 in two; 64 of one and four of 64 behind 8192, 183 and 43 + 58; 30 of one and
    // two of 512 behind 2048, 86 and 26 + 64. A caller who passes a max_query of 64 rows gets phases: 509, 85 and 93 us.
    const int64_t group_rows = groups > 0 ? tokens * share / groups : 0;
    if (groups > 0 && group_rows > row_rows && row_rows <= 64) {
        plan.pair = true;
        plan.tiles16 = row_rows <= 16 ? 1 : 8;
        cut(plan, plan.own, kOwn, batch, plan.tiles16, tokens, share, kv_heads, dim_pad, false);
        cut(plan, plan.prefix, kPrefixes, groups, 8, tokens, share, kv_heads, dim_pad, false);
    } else {
        plan.tiles16 = tiles_for(row_rows, dim_pad);
        cut(plan, plan.own, groups > 0 ? kWhole : kOwn, batch, plan.tiles16, tokens, share, kv_heads, dim_pad, true);
    }
    return plan;
}

Plan topk_plan(int64_t tokens, int64_t lanes, int64_t heads, int64_t kv_heads, int64_t dim) {
    if (lanes < 0) {
        throw std::invalid_argument("the number of lanes is negative");
    }
    need_sizes(tokens, 0, heads, kv_heads, dim);
    Plan plan;
    plan.tiles16 = tiles_for(heads / kv_heads, padded_dim(dim));
    cut(plan, plan.own, kSlots, tokens, plan.tiles16, tokens, heads / kv_heads, kv_heads, padded_dim(dim), true);
    return plan;
}

Plan block_plan(int64_t tokens, int64_t width, int64_t block_size, int64_t heads, int64_t kv_heads, int64_t dim,
                int64_t max_query) {
    constexpr int64_t kMost = (int64_t{1} << 30) - 1;
    if (block_size < 1 || block_size > kMost || width < 0 || width > kMost / block_size) {
        throw std::invalid_argument("a list of blocks may name at most 2^30 - 1 tokens");
    }
    if (max_query < 1) {
        throw std::invalid_argument("max_query must be positive");
    }
    need_sizes(tokens, 0, heads, kv_heads, dim);
    Plan plan;
    const int32_t dim_pad = padded_dim(dim);
    // 64 tokens' 32 blocks of 64, one KV head of 128, by 1, 2 and 4 row tiles: 16 query heads 24, 25 and 30 us, 32 heads 34,
    // 26 and 31, 64 heads 54, 38 and 34; of 256, where two spill 76 registers, by 1 and 2: 32 heads 57 and 59, 64 heads
    // 97 and 91.
    plan.tiles16 = dim_pad <= 128 ? std::min(tiles_for(heads / kv_heads, dim_pad), 4) : 1;
    cut(plan, plan.own, kSlots, tokens, plan.tiles16, tokens, heads / kv_heads, kv_heads, dim_pad, true);
    return plan;
}

void place(Phase& p, void* workspace) {
    const auto at = [&](auto*& pointer) {
        pointer = reinterpret_cast<std::remove_reference_t<decltype(pointer)>>(static_cast<char*>(workspace) +
                                                                              reinterpret_cast<uintptr_t>(pointer));
    };
    at(p.parts);
    if (p.mode != kSlots) {
        at(p.unit_starts);
        at(p.item_starts);
    }
}

void need_workspace(const Plan& plan, const void* workspace, uint64_t bytes) {
    if (bytes < plan.bytes) {
        throw std::invalid_argument("the attention needs " + std::to_string(plan.bytes) + " workspace bytes, got " +
                                    std::to_string(bytes));
    }
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0) {
        throw std::invalid_argument("the workspace must be a 256-byte aligned device buffer");
    }
}

int launch(const AttentionArgs& a, Plan& plan, int32_t dtype, void* workspace, uint64_t bytes, void* stream,
           const BlockLists* lists = nullptr) {
    need_workspace(plan, workspace, bytes);
    if (a.tokens == 0) {
        return 0;
    }
    place(plan.own, workspace);
    fit_units(plan.own, int64_t{a.own_most} + a.prefix_most);
    if (plan.own.mode == kSlots) {
        Phase& p = plan.own;
        const int64_t units = std::max<int64_t>((int64_t{a.own_most} + (1 << p.unit_shift) - 1) >> p.unit_shift, 1);
        const int64_t items = int64_t{a.kv_heads} * ((a.share + (1 << p.row_shift) - 1) >> p.row_shift);
        p.alike_units = FastDiv(static_cast<uint32_t>(units));
        p.alike_items = FastDiv(static_cast<uint32_t>(items));
        p.alike_total = static_cast<uint32_t>(units * items * a.tokens);
    }
    if (plan.pair) {
        place(plan.prefix, workspace);
        fit_units(plan.prefix, a.prefix_most);
        launch_pair(Launch{a, {plan.own, plan.prefix}, {}}, dtype, stream);
    } else if (lists != nullptr) {
        launch_blocks(Launch{a, {plan.own, {}}, *lists}, dtype, plan.tiles16, stream);
    } else if (plan.tiles16 < 8) {
        launch_narrow(Launch{a, {plan.own, {}}, {}}, dtype, plan.tiles16, stream);
    } else {
        launch_wide(Launch{a, {plan.own, {}}, {}}, dtype, stream);
    }
    const auto merge = [&]<typename T>(T) {
        const auto on = static_cast<hipStream_t>(stream);
        // By tokens the time goes with the rows, by cuts with the workgroups: a whole call of 64, 256, 512 and 2048
        // tokens of 8 KV heads takes 25, 80, 155 and 583 us by tokens and 29, 81, 153 and 550 by cuts; eight prompts'
        // pieces of up to 1024 tokens take 62 us more by tokens and 22 by cuts.
        if (!plan.pair && int64_t{a.tokens} * a.kv_heads > kComputeUnits * kMergeByToken) {
            const dim3 grid(plan.own.workgroups, kMergeColumns);
            cuts_kernel<T><<<grid, kMergeThreads, 0, on>>>(a, plan.own);
        } else {
            const uint32_t pieces = (a.share * ((a.dim + 3) / 4) + kMergeThreads - 1) / kMergeThreads;
            const dim3 grid(static_cast<uint32_t>(a.tokens), static_cast<uint32_t>(a.kv_heads),
                            std::min(pieces, uint32_t{64}));
            merge_kernel<T><<<grid, kMergeThreads, 0, on>>>(a, plan.own, plan.prefix);
        }
    };
    if (dtype == EKV_BFLOAT16) {
        merge(Bf16{});
    } else {
        merge(F16{});
    }
    check_hip(hipGetLastError(), "launch attention merge");
    return 0;
}

const ekv_tensor& need_table(const ekv_tensor* p, int64_t page_size, const char* name) {
    const ekv_tensor& t = need(p, name);
    need_ndim(t, 2, name);
    need_index(t, name);
    need_data(t, name);
    if (t.shape[1] > ((int64_t{1} << 30) - 1) / page_size) {
        throw std::invalid_argument(std::string(name) + " rows may cover at most 2^30 - 1 tokens");
    }
    return t;
}

// The batch rows: their pages, lengths and query tokens. Returns how many tokens a table row covers.
int32_t own_tables(AttentionArgs& a, const ekv_tensor* tables_p, const ekv_tensor* rows, const ekv_tensor* lengths_p,
                   const ekv_tensor* query_starts, int64_t max_query, int64_t page_size) {
    const ekv_tensor& tables = need_table(tables_p, page_size, "block_tables");
    const ekv_tensor& lengths = need(lengths_p, "lengths");
    need_ndim(lengths, 1, "lengths");
    need_index(lengths, "lengths");
    need_data(lengths, "lengths");
    if (lengths.shape[0] > kMostBatch) {
        throw std::invalid_argument("more than 2^20 batch rows");
    }
    a.batch = static_cast<int32_t>(lengths.shape[0]);
    a.lengths = index_ref(lengths, 0);
    a.tables = static_cast<const char*>(tables.data);
    a.table_row = tables.stride[0] * itemsize(tables.dtype);
    a.table_col = column_step(tables, "block_tables");
    a.table64 = tables.dtype == EKV_INT64;
    a.requests = static_cast<int32_t>(std::min<int64_t>(tables.shape[0], 0x7fffffff));
    if (rows != nullptr) {
        a.rows = index_ref(need_list(rows, a.batch, "rows"), 0);
    }
    if (max_query < 1) {
        throw std::invalid_argument("max_query must be positive");
    }
    if (query_starts != nullptr) {
        a.query_starts = index_ref(need_list(query_starts, a.batch + 1, "query_starts"), 0);
    } else if (a.tokens != a.batch) {
        throw std::invalid_argument("without query_starts every batch row has one query token: got " +
                                    std::to_string(a.tokens) + " for " + std::to_string(a.batch) + " rows");
    }
    return static_cast<int32_t>(tables.shape[1] * page_size);
}

int shared_prefix(const ekv_prefix_attention_args& s, void* workspace, uint64_t workspace_bytes, void* stream) {
    AttentionArgs a = common_args(s.query, s.planes, s.layer, s.kv_heads, s.page_size, s.scale, s.output, s.lse);
    a.own_most = own_tables(a, s.block_tables, s.rows, s.lengths, s.query_starts, s.max_query, s.page_size);
    if ((s.prefix_tables == nullptr) != (s.prefix_lengths == nullptr)) {
        throw std::invalid_argument("prefix_tables and prefix_lengths are given together");
    }
    if (s.prefix_tables != nullptr) {
        const ekv_tensor& prefix = need_table(s.prefix_tables, s.page_size, "prefix_tables");
        if (prefix.shape[0] > kMostBatch) {
            throw std::invalid_argument("more than 2^20 prefixes");
        }
        a.groups = static_cast<int32_t>(prefix.shape[0]);
        a.prefix_tables = static_cast<const char*>(prefix.data);
        a.prefix_row = prefix.stride[0] * itemsize(prefix.dtype);
        a.prefix_col = column_step(prefix, "prefix_tables");
        a.prefix64 = prefix.dtype == EKV_INT64;
        a.prefix_most = static_cast<int32_t>(prefix.shape[1] * s.page_size);
        a.prefix_lengths = index_ref(need_list(s.prefix_lengths, a.groups, "prefix_lengths"), 0);
        if (s.group_starts != nullptr) {
            a.group_starts = index_ref(need_list(s.group_starts, a.groups + 1, "group_starts"), 0);
        } else if (a.groups > 1) {
            throw std::invalid_argument("more than one prefix needs group_starts");
        }
    } else if (s.group_starts != nullptr) {
        throw std::invalid_argument("group_starts without prefix_tables");
    }
    Plan plan = prefix_plan(a.tokens, a.batch, a.groups, a.heads, a.kv_heads, a.dim, s.max_query);
    return launch(a, plan, s.query->dtype, workspace, workspace_bytes, stream);
}

int topk(const ekv_tensor* query, const ekv_planes* planes, int64_t layer, int64_t kv_heads, const ekv_tensor* slots_p,
         int64_t zero_below, double scale, const ekv_tensor* out, const ekv_tensor* lse, void* workspace,
         uint64_t workspace_bytes, void* stream) {
    AttentionArgs a = common_args(query, planes, layer, kv_heads, 1, scale, out, lse);
    const ekv_tensor& slots = need(slots_p, "slots");
    need_ndim(slots, 2, "slots");
    need_index(slots, "slots");
    need_dim(slots, 0, a.tokens, "slots");
    need_data(slots, "slots");
    if (slots.shape[1] > (int64_t{1} << 30) - 1) {
        throw std::invalid_argument("more than 2^30 - 1 lanes");
    }
    if (zero_below < 0 || zero_below > 0x7fffffff) {
        throw std::invalid_argument("zero_below must be from 0 to 2^31 - 1");
    }
    a.cache.zero_below = static_cast<uint32_t>(zero_below);
    a.batch = a.tokens;
    a.tables = static_cast<const char*>(slots.data);
    a.table_row = slots.stride[0] * itemsize(slots.dtype);
    a.table_col = column_step(slots, "slots");
    a.table64 = slots.dtype == EKV_INT64;
    a.requests = a.tokens;
    a.own_most = static_cast<int32_t>(slots.shape[1]);
    Plan plan = topk_plan(a.tokens, a.own_most, a.heads, a.kv_heads, a.dim);
    return launch(a, plan, query->dtype, workspace, workspace_bytes, stream);
}

// Whether query tokens go through their lists together: where batch rows fill tiles of 64 rows, and where the kernel for few
// rows would have so many (token, KV head) pairs that its time passes that of a workgroup's blocks one after the other.
// Lists of 16 blocks of 64 behind 16384 tokens, neighbours' alike, together and one by one: 16 heads on 2 of 128, four
// pieces of 256 tokens 78 and 141 us, eight of 64 (1024 pairs) 76 and 76, one of 256 83 and 41; 32 heads on 4 of 128,
// eight of 64 80 and 142, eight of 32 78 and 76; 8 heads on 8 of 64, eight of 64 (4096 pairs of half the bytes) 67 and 149,
// eight of 32 67 and 87. The host cannot see whether they are alike: random lists take 178 and 144, 188 and 84, 181 and
// 42; 219 and 154, 179 and 83; 328 and 154, 288 and 90. Blocks go in runs of 32 keys, the last part-filled: eight pieces of
// 128 tokens (2048 pairs) of 16 heads on 2 of 128 with 16 blocks of 100 take 114 and 206 us, with 32 of 20 77 and 100, with
// 32 of 16 80 and 87. At a head size of 256, eight of 128 take 172 and 305, eight of 64 175 and 157.
bool union_pays(const AttentionArgs& a, const BlockLists& lists, int64_t block_size, int64_t max_query, int32_t dim_pad) {
    const int64_t tile_tokens = std::min<int64_t>(64, 63 / a.share + 2);
    // Without batch rows there may be no tile, and lists of no entries have no width to divide by: the other kernel writes
    // the zeros.
    const bool fits = a.batch > 0 && lists.width > 0 && block_size >= 16 &&
                      tile_tokens * lists.width <= kUnionEntries && a.block_most / block_size < kUnionBlocks &&
                      (int64_t{a.tokens} * a.share / 64 + a.batch) * a.kv_heads < 1 << 24;   // fewer than 2^32 threads
    const int64_t filled = (block_size + 31) / 32 * 32;
    const int64_t pairs = int64_t{a.tokens} * a.kv_heads * std::min(dim_pad, 128) / 128 * block_size / filled;
    return fits && a.share <= 32 && max_query * a.share >= 64 && pairs >= 2048;
}

int block_attention(const ekv_block_attention_args& s, void* workspace, uint64_t workspace_bytes, void* stream) {
    AttentionArgs a = common_args(s.query, s.planes, s.layer, s.kv_heads, s.page_size, s.scale, s.output, s.lse);
    a.block_most = own_tables(a, s.block_tables, s.rows, s.lengths, s.query_starts, s.max_query, s.page_size);
    const ekv_tensor& blocks = need(s.blocks, "blocks");
    need_ndim(blocks, 3, "blocks");
    need_index(blocks, "blocks");
    need_dim(blocks, 0, a.tokens, "blocks");
    need_data(blocks, "blocks");
    if (blocks.shape[1] < 1 || a.kv_heads % blocks.shape[1] != 0) {
        throw std::invalid_argument("blocks must have a divisor of kv_heads as lists");
    }
    Plan plan = block_plan(a.tokens, blocks.shape[2], s.block_size, a.heads, a.kv_heads, a.dim, s.max_query);
    a.own_most = static_cast<int32_t>(blocks.shape[2] * s.block_size);
    BlockLists lists{};
    lists.lists = static_cast<const char*>(blocks.data);
    lists.token = blocks.stride[0] * itemsize(blocks.dtype), lists.group = blocks.stride[1] * itemsize(blocks.dtype);
    lists.column = column_step(blocks, "blocks", 2);
    lists.wide = blocks.dtype == EKV_INT64 ? 4 : 0;
    lists.block = FastDiv(static_cast<uint32_t>(s.block_size));
    lists.heads = FastDiv(static_cast<uint32_t>(a.kv_heads / blocks.shape[1]));
    lists.width = static_cast<int32_t>(blocks.shape[2]);
    need_distinct(*s.output, "output");
    if (!same_view(*s.query, *s.output)) {
        need_apart(Extent(s.output), "output", Extent(s.query), "query, unless it is the query");
    }
    const PlanePages pages = plane_pages(s.planes, s.layer, int64_t{a.kv_heads} * a.dim * 2, s.page_size, 2);
    const Extent planes[2] = {Extent(pages, *s.planes, 0), Extent(pages, *s.planes, 1)};
    const auto apart = [&](const Extent& e, const char* name) {
        for (const Extent& plane : planes) {
            need_apart(e, name, plane, "the layer's planes");
        }
        need_apart(e, name, Extent(s.block_tables), "block_tables");
        need_apart(e, name, Extent(s.rows), "rows");
        need_apart(e, name, Extent(s.lengths), "lengths");
        need_apart(e, name, Extent(&blocks), "blocks");
        need_apart(e, name, Extent(s.query_starts), "query_starts");
    };
    apart(Extent(s.output), "output");
    if (s.lse != nullptr) {
        need_distinct(*s.lse, "lse");
        apart(Extent(s.lse), "lse");
        need_apart(Extent(s.lse), "lse", Extent(s.query), "query");
        need_apart(Extent(s.lse), "lse", Extent(s.output), "output");
    }
    need_workspace(plan, workspace, workspace_bytes);
    const Extent work(workspace, plan.bytes);
    apart(work, "the workspace");
    need_apart(work, "the workspace", Extent(s.query), "query");
    need_apart(work, "the workspace", Extent(s.output), "output");
    need_apart(work, "the workspace", Extent(s.lse), "lse");
    if (s.query_starts != nullptr && union_pays(a, lists, s.block_size, s.max_query, plan.own.dim_pad)) {
        if (a.tokens > 0) {
            lists.runs_of = FastDiv(static_cast<uint32_t>((s.block_size + 31) / 32));
            lists.tiles = static_cast<int32_t>(int64_t{a.tokens} * a.share / 64 + a.batch);
            launch_union(Launch{a, {plan.own, {}}, lists}, s.query->dtype, stream);
        }
        return 0;
    }
    return launch(a, plan, s.query->dtype, workspace, workspace_bytes, stream, &lists);
}

}  // namespace
}  // namespace ekv

extern "C" uint64_t ekv_shared_prefix_workspace_bytes(int64_t tokens, int64_t batch, int64_t groups, int64_t heads,
                                                      int64_t kv_heads, int64_t head_dim, int64_t max_query) {
    return ekv::guarded(~uint64_t{0}, [&] {
        return ekv::prefix_plan(tokens, batch, groups, heads, kv_heads, head_dim, max_query).bytes;
    });
}

extern "C" int ekv_shared_prefix_attention(const ekv_prefix_attention_args* args, void* workspace,
                                           uint64_t workspace_bytes, void* stream) {
    return ekv::guarded(-1, [&] {
        if (args == nullptr) {
            throw std::invalid_argument("args is required");
        }
        return ekv::shared_prefix(*args, workspace, workspace_bytes, stream);
    });
}

extern "C" uint64_t ekv_topk_workspace_bytes(int64_t tokens, int64_t lanes, int64_t heads, int64_t kv_heads,
                                             int64_t head_dim) {
    return ekv::guarded(~uint64_t{0}, [&] { return ekv::topk_plan(tokens, lanes, heads, kv_heads, head_dim).bytes; });
}

extern "C" int ekv_topk_attention(const ekv_tensor* query, const ekv_planes* planes, int64_t layer, int64_t kv_heads,
                                  const ekv_tensor* slots, int64_t zero_below, double scale, const ekv_tensor* output,
                                  const ekv_tensor* lse, void* workspace, uint64_t workspace_bytes, void* stream) {
    return ekv::guarded(-1, [&] {
        return ekv::topk(query, planes, layer, kv_heads, slots, zero_below, scale, output, lse, workspace,
                         workspace_bytes, stream);
    });
}

extern "C" uint64_t ekv_block_workspace_bytes(int64_t tokens, int64_t width, int64_t block_size, int64_t heads,
                                              int64_t kv_heads, int64_t head_dim, int64_t max_query) {
    return ekv::guarded(~uint64_t{0}, [&] {
        return ekv::block_plan(tokens, width, block_size, heads, kv_heads, head_dim, max_query).bytes;
    });
}

extern "C" int ekv_block_attention(const ekv_block_attention_args* args, void* workspace, uint64_t workspace_bytes,
                                   void* stream) {
    return ekv::guarded(-1, [&] {
        if (args == nullptr) {
            throw std::invalid_argument("args is required");
        }
        return ekv::block_attention(*args, workspace, workspace_bytes, stream);
    });
}
