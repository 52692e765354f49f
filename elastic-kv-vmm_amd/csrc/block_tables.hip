// Block tables and slot maps of a serving step, built from request lengths (gfx950).
//
// Every batch row b holds len_b tokens in pages of p tokens and gets add_b more:
//   have_b = ceil(len_b / p), need_b = ceil((len_b + add_b) / p)
//   base_b = sum over earlier rows of (need - have), start_b = sum over earlier rows of add
//   table[rows_b, j]   = free[head + base_b + j - have_b]                 have_b <= j < need_b
//   slots[start_b + i] = table[rows_b, (len_b + i) / p] * p + (len_b + i) % p,  position len_b + i
// Both sums are taken by every workgroup for itself (a few loads and two DPP scans per 1024 rows), so one launch does
// it all with no workgroup waiting for another: a new page's id is read from the free list, never from the table that
// another workgroup may be writing, and table entries below have_b are written by nobody.
//
// What bounds it: for a decode step the chain of launch, lengths, sums, table entry, store, 9.5 us for 128 requests (a
// launch of an empty kernel and four dependent memory levels); for long prompts the stores behind that chain, 38 MB of
// slots and positions of 251 requests in 21 us. There a thread's four tokens share one lookup (24 us when each had its
// own), and 1024 workgroups take tiles of 1024 tokens in turn: 256, 512, 768 and 1536 take 37, 26, 22 and 25 us.
#include "../../include/ekv_kernels.h"
#include "ekv_common.h"
#include "ekv_fastdiv.h"
#include "ekv_tensor_util.h"
#include "ekv_vec.h"
#include "ekv_wave.h"

#include <algorithm>
#include <limits>
#include <numeric>

namespace ekv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kPer = 4;                        // rows per thread of a chunk
constexpr int kChunk = kThreads * kPer;        // rows whose sums a workgroup holds at a time
constexpr int kTokens = 4;                     // tokens per thread and step: one 16-byte store of int32 slots
constexpr int kTile = kThreads * kTokens;
constexpr int64_t kMaxGroups = 1024;           // four a compute unit

// An int32 or int64 array that is written.
struct IndexOut {
    void* data = nullptr;
    int64_t stride = 0;
    int32_t is64 = 0;

    __device__ __forceinline__ void put(int64_t i, int64_t value) const {
        if (is64) {
            static_cast<int64_t*>(data)[i * stride] = value;
        } else {
            static_cast<int32_t*>(data)[i * stride] = static_cast<int32_t>(value);
        }
    }
};

struct TableArgs {
    void* table;
    int64_t table_row, table_col;
    int64_t requests, columns;
    int32_t table64;
    IndexRef rows, lengths, added, free_pages, free_head;
    IndexOut slots, positions, starts, new_lengths, new_head;
    int32_t has_positions, vector;
    int64_t batch, capacity, free_count, page_size;
    int64_t most_id;              // the largest page id whose slots are below 2^63
    FastDiv page;
    int32_t* status;
};

// Exclusive sum over the workgroup of one value below 2^32 per thread: the low 20 bits and the others are scanned
// apart, so that neither sum of 256 values leaves 32 bits.
__device__ __forceinline__ int64_t workgroup_before(int64_t value, uint32_t (*cells)[kWaves], int64_t& total) {
    const uint32_t low = static_cast<uint32_t>(value) & 0xfffffu;
    const uint32_t high = static_cast<uint32_t>(value >> 20);
    const uint32_t low_sum = wave_scan<kAdd>(low), high_sum = wave_scan<kAdd>(high);
    const int wave = threadIdx.x >> 6;
    __syncthreads();   // the cells' last use
    if ((threadIdx.x & 63) == 63) {
        cells[0][wave] = low_sum;
        cells[1][wave] = high_sum;
    }
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const int64_t sum = static_cast<int64_t>(cells[0][w]) + (static_cast<int64_t>(cells[1][w]) << 20);
        before += w < wave ? sum : 0;
        total += sum;
    }
    return before + static_cast<int64_t>(low_sum - low) + (static_cast<int64_t>(high_sum - high) << 20);
}

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// The page id at place `from` of the free list: 0, the sink, past the list's ends and for an id that the table's type
// cannot hold (its low half could name another page).
__device__ __forceinline__ int64_t new_page(const TableArgs& a, int64_t from, int32_t& flags) {
    const int64_t id = from >= 0 && from < a.free_count ? a.free_pages[from] : 0;
    const bool fits = a.table64 || id == static_cast<int32_t>(id);
    flags |= fits ? 0 : EKV_TABLES_ID_RANGE;
    return fits ? id : 0;
}

// The first slot of a row's page `column`, -1 for none: a page that the row had is in its table, a new one in the list.
__device__ __forceinline__ int64_t page_slot(const TableArgs& a, int64_t head, int64_t row, int64_t base, uint32_t column,
                                             uint32_t held, int32_t& flags) {
    int64_t id;
    if (column < held) {
        const int64_t entry = row * a.table_row + int64_t{column} * a.table_col;
        id = a.table64 ? static_cast<const int64_t*>(a.table)[entry] : static_cast<const int32_t*>(a.table)[entry];
    } else {
        id = new_page(a, head + base + (column - held), flags);
    }
    flags |= id > a.most_id ? EKV_TABLES_SLOT_RANGE : 0;
    return id >= 1 && id <= a.most_id ? id * a.page_size : -1;
}

// The last of entries low .. high - 1 that is at most `value` (entry `low` is).
__device__ __forceinline__ int last_not_above(const int64_t* entries, int low, int high, int64_t value) {
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (entries[mid] <= value) {
            low = mid;
        } else {
            high = mid;
        }
    }
    return low;
}

// The same among the first `count` entries for a value that a wave shares: its lanes look at 64 entries at a time.
__device__ __forceinline__ int wave_last_not_above(const int64_t* entries, int count, int64_t value) {
    const int lane = threadIdx.x & 63, step = (count + 63) >> 6;
    const int coarse = lane * step;
    const int base = (__popcll(__ballot(coarse < count && entries[min(coarse, count - 1)] <= value)) - 1) * step;
    const int fine = base + lane;
    return base + __popcll(__ballot(lane < step && fine < count && entries[min(fine, count - 1)] <= value)) - 1;
}

// The kernel's arguments. They are more words than a wave has scalar registers: hidden from the compiler where they come
// from, each part of the kernel loads what it needs, instead of one load of all and spills.
__device__ __forceinline__ const TableArgs& arguments() {
    auto at = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const TableArgs*)(at);
}

__global__ __launch_bounds__(kThreads) void extend_tables_kernel(const TableArgs) {
    __shared__ int64_t s_start[kChunk];    // first token of each row of the chunk
    __shared__ int64_t s_base[kChunk];     // first new page of each row
    __shared__ int32_t s_length[kChunk], s_row[kChunk];
    __shared__ uint32_t s_cells[2][kWaves];
    const int tid = threadIdx.x;
    const bool first = blockIdx.x == 0;
    const int64_t head = arguments().free_head.fetch(0);
    const int64_t batch = arguments().batch;
    int64_t token_base = 0, page_base = 0;
    int32_t flags = 0;

    for (int64_t chunk = 0; chunk < batch; chunk += kChunk) {
        const int count = static_cast<int>(min(static_cast<int64_t>(kChunk), batch - chunk));
        const TableArgs& a = arguments();
        const int64_t room = a.columns * a.page_size;
        // Thread t sums rows t * kPer .. + kPer - 1 of the chunk; what it knows of each waits in its places in LDS.
        int64_t token_sum = 0, page_sum = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int at = tid * kPer + k;
            const bool live = at < count;
            const int64_t b = chunk + (live ? at : 0);
            const int64_t length = a.lengths.fetch(b), added = a.added.fetch(b);
            const int64_t given = (a.rows.data != nullptr ? a.rows : a.lengths).fetch(b);   // in flight with the others
            const int64_t row = a.rows.data != nullptr ? given : b;
            const bool good = row >= 0 && row < a.requests && length >= 0 && length <= room && added >= 0;
            const int64_t held = live ? min(max(length, int64_t{0}), room) : 0;
            const int64_t fits = live && good ? min(added, room - held) : 0;
            flags |= good ? 0 : EKV_TABLES_BAD_ROW;
            flags |= live && good && added > fits ? EKV_TABLES_ROW_FULL : 0;
            const uint32_t held_pages = a.page.div(static_cast<uint32_t>(held) + a.page.divisor - 1);
            const uint32_t need_pages = a.page.div(static_cast<uint32_t>(held + fits) + a.page.divisor - 1);
            s_start[at] = fits;
            s_base[at] = need_pages - held_pages;
            s_length[at] = static_cast<int32_t>(held);
            s_row[at] = good ? static_cast<int32_t>(row) : 0;
            token_sum += fits;
            page_sum += need_pages - held_pages;
        }
        // A row adds fewer than 2^30 tokens, a thread's four fewer than 2^32.
        int64_t token_total = 0, page_total = 0;
        int64_t token_at = token_base + workgroup_before(token_sum, s_cells, token_total);
        int64_t page_at = page_base + workgroup_before(page_sum, s_cells, page_total);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int at = tid * kPer + k;
            const int64_t fits = s_start[at], pages = s_base[at];
            s_start[at] = token_at;
            s_base[at] = page_at;
            if (first && at < count) {
                a.starts.put(chunk + at, min(token_at, a.capacity));
                a.new_lengths.put(chunk + at, s_length[at] + fits);
            }
            token_at += fits;
            page_at += pages;
        }
        __syncthreads();

        // The chunk's new pages.
        const int64_t page_end = page_base + page_total;
        for (int64_t u = page_base + int64_t{blockIdx.x} * kThreads + tid; u < page_end;
             u += int64_t{gridDim.x} * kThreads) {
            const int r = last_not_above(s_base, 0, count, u);
            const int64_t id = new_page(a, head + u, flags);
            const uint32_t held = a.page.div(static_cast<uint32_t>(s_length[r]) + a.page.divisor - 1);
            const int64_t at = s_row[r] * a.table_row + (held + (u - s_base[r])) * a.table_col;
            if (a.table64) {
                static_cast<int64_t*>(a.table)[at] = id;
            } else {
                static_cast<int32_t*>(a.table)[at] = static_cast<int32_t>(id);
            }
        }

        // The chunk's tokens: tiles of the whole map, so that a thread's four slots are one aligned store.
        const int64_t token_end = min(token_base + token_total, a.capacity);
        int64_t tile = token_base / kTile;
        tile += (int64_t{blockIdx.x} + gridDim.x - tile % gridDim.x) % gridDim.x;
        for (; tile * kTile < token_end; tile += gridDim.x) {
            const int64_t t = tile * kTile + tid * kTokens;
            // Rows of the wave's first and last token: long rows leave each lane little to search.
            const int64_t wave_first = max(tile * kTile + (tid & ~63) * kTokens, token_base);
            const int64_t wave_last = min(tile * kTile + (tid | 63) * kTokens + kTokens, token_end) - 1;
            if (wave_first > wave_last) {
                continue;
            }
            const int row_first = wave_last_not_above(s_start, count, wave_first);
            const int row_last = wave_last_not_above(s_start, count, wave_last);
            int r = t >= token_base && t < token_end ? last_not_above(s_start, row_first, row_last + 1, t) : 0;
            const bool whole = t >= token_base && t + kTokens <= token_end;
            if (a.vector && whole && a.page_size >= kTokens &&
                (r + 1 < count ? s_start[r + 1] : token_end) >= t + kTokens) {
                // Four tokens of one row, on one page or two.
                const uint32_t length = static_cast<uint32_t>(s_length[r]);
                const uint32_t position = length + static_cast<uint32_t>(t - s_start[r]);
                const uint32_t column = a.page.div(position), offset = position - column * a.page.divisor;
                const bool crosses = offset + kTokens > a.page.divisor;
                const uint32_t held = a.page.div(length + a.page.divisor - 1);
                const int64_t page = page_slot(a, head, s_row[r], s_base[r], column, held, flags);
                int64_t next = page;
                if (crosses) {
                    next = page_slot(a, head, s_row[r], s_base[r], column + 1, held, flags);
                }
                i32x4 slot, place;
#pragma unroll
                for (int k = 0; k < kTokens; ++k) {
                    const bool here = offset + k < a.page.divisor;
                    const int64_t first_slot = here ? page : next;
                    const int64_t value = first_slot + (here ? offset + k : offset + k - a.page.divisor);
                    const bool fits = value <= 0x7fffffff;
                    flags |= first_slot >= 0 && !fits ? EKV_TABLES_SLOT_RANGE : 0;
                    slot[k] = first_slot >= 0 && fits ? static_cast<int32_t>(value) : -1;
                    place[k] = static_cast<int32_t>(position + k);
                }
                *reinterpret_cast<i32x4*>(static_cast<int32_t*>(a.slots.data) + t) = slot;
                if (a.has_positions) {
                    *reinterpret_cast<i32x4*>(static_cast<int32_t*>(a.positions.data) + t) = place;
                }
                continue;
            }
            int32_t slot32[kTokens], position32[kTokens];
#pragma unroll
            for (int k = 0; k < kTokens; ++k) {
                const int64_t at = t + k;
                if (at < token_base || at >= token_end) {
                    continue;
                }
                while (r + 1 < count && s_start[r + 1] <= at) {
                    ++r;
                }
                const uint32_t length = static_cast<uint32_t>(s_length[r]);
                const uint32_t position = length + static_cast<uint32_t>(at - s_start[r]);
                const uint32_t column = a.page.div(position);
                const uint32_t held = a.page.div(length + a.page.divisor - 1);
                const int64_t page = page_slot(a, head, s_row[r], s_base[r], column, held, flags);
                int64_t slot = page >= 0 ? page + (position - column * a.page.divisor) : -1;
                if (!a.slots.is64 && slot > 0x7fffffff) {
                    flags |= EKV_TABLES_SLOT_RANGE;
                    slot = -1;
                }
                if (a.vector) {
                    slot32[k] = static_cast<int32_t>(slot);
                    position32[k] = static_cast<int32_t>(position);
                }
                if (!a.vector || !whole) {
                    a.slots.put(at, slot);
                    if (a.has_positions) {
                        a.positions.put(at, position);
                    }
                }
            }
            if (a.vector && whole) {
                *reinterpret_cast<i32x4*>(static_cast<int32_t*>(a.slots.data) + t) =
                    i32x4{slot32[0], slot32[1], slot32[2], slot32[3]};
                if (a.has_positions) {
                    *reinterpret_cast<i32x4*>(static_cast<int32_t*>(a.positions.data) + t) =
                        i32x4{position32[0], position32[1], position32[2], position32[3]};
                }
            }
        }
        token_base += token_total;
        page_base = page_end;
        __syncthreads();   // the chunk's sums are read before the next chunk's replace them
    }

    const TableArgs& a = arguments();
    // Places of the map that no token has.
    for (int64_t t = token_base + int64_t{blockIdx.x} * kThreads + tid; t < a.capacity;
         t += int64_t{gridDim.x} * kThreads) {
        a.slots.put(t, -1);
        if (a.has_positions) {
            a.positions.put(t, -1);
        }
    }
    if (first && tid == 0) {
        a.starts.put(a.batch, min(token_base, a.capacity));
        a.new_head.put(0, head + page_base);
        if (token_base > a.capacity) {
            flags |= EKV_TABLES_MAP_FULL;
        }
        if (head < 0 || (page_base > 0 && head > a.free_count - page_base)) {
            flags |= EKV_TABLES_NO_PAGES;
        }
    }
    if (flags != 0 && a.status != nullptr) {
        atomicOr(a.status, flags);
    }
}

const ekv_tensor& need_vector(const ekv_tensor* p, int64_t extent, const char* name) {
    const ekv_tensor& t = need(p, name);
    need_ndim(t, 1, name);
    need_index(t, name);
    if (extent >= 0) {
        need_dim(t, 0, extent, name);
    }
    need_data(t, name);
    return t;
}

IndexOut index_out(const ekv_tensor& t) {
    IndexOut out;
    out.data = t.data;
    out.stride = t.stride[0];
    out.is64 = t.dtype == EKV_INT64;
    return out;
}

// The bytes of a one-dimensional array: from `begin` to `end`, elements of `item` bytes `step` apart.
struct Bytes {
    int64_t begin = 0, end = 0, step = 0, item = 0;

    explicit Bytes(const ekv_tensor* t) {
        if (t == nullptr || t->shape[0] == 0) {
            return;
        }
        item = itemsize(t->dtype);
        step = t->shape[0] > 1 ? t->stride[0] * item : 0;
        const int64_t first = static_cast<int64_t>(reinterpret_cast<uintptr_t>(t->data));
        const int64_t last = first + (t->shape[0] - 1) * step;
        begin = std::min(first, last);
        end = std::max(first, last) + item;
    }

    // Whether the arrays may share a byte. Their elements lie at whole multiples of the strides' greatest common divisor
    // from each other, so arrays that lie in one another without a shared element, as columns of one tensor, are told
    // apart.
    bool meets(const Bytes& other) const {
        if (item == 0 || other.item == 0 || begin >= other.end || other.begin >= end) {
            return false;
        }
        const int64_t common = std::gcd(step, other.step);
        if (common == 0) {
            return true;
        }
        const int64_t apart = ((other.begin - begin) % common + common) % common;
        return apart < item || common - apart < other.item;
    }
};

int extend_block_tables(const ekv_tensor* table_p, const ekv_tensor* rows_p, const ekv_tensor* lengths_p,
                        const ekv_tensor* added_p, const ekv_tensor* free_p, const ekv_tensor* head_p,
                        int64_t page_size, const ekv_tensor* slots_p, const ekv_tensor* positions_p,
                        const ekv_tensor* starts_p, const ekv_tensor* new_lengths_p, const ekv_tensor* new_head_p,
                        const ekv_tensor* status_p, void* stream) {
    const ekv_tensor& table = need(table_p, "block_tables");
    need_ndim(table, 2, "block_tables");
    need_index(table, "block_tables");
    need_data(table, "block_tables");
    if (page_size < 1) {
        throw std::invalid_argument("page_size must be positive");
    }
    // Positions are 31-bit: page_size <= 2^31 - 1 is checked first, so the product cannot wrap.
    constexpr int64_t kMost = (int64_t{1} << 30) - 1;
    if (page_size > kMost || table.shape[1] > kMost / page_size || table.shape[0] > 0x7fffffff) {
        throw std::invalid_argument("a block table row may cover at most 2^30 - 1 tokens");
    }
    const ekv_tensor& lengths = need_vector(lengths_p, -1, "lengths");
    const int64_t batch = lengths.shape[0];
    const ekv_tensor& added = need_vector(added_p, batch, "added");
    const ekv_tensor& free_pages = need_vector(free_p, -1, "free_pages");
    const ekv_tensor& head = need_vector(head_p, 1, "free_head");
    const ekv_tensor& slots = need_vector(slots_p, -1, "slots");
    const ekv_tensor& starts = need_vector(starts_p, batch + 1, "starts");
    const ekv_tensor& new_lengths = need_vector(new_lengths_p, batch, "new_lengths");
    const ekv_tensor& new_head = need_vector(new_head_p, 1, "new_head");
    constexpr int64_t kMost32 = std::numeric_limits<int32_t>::max();
    if ((starts.dtype == EKV_INT32 && slots.shape[0] > kMost32) ||
        (new_head.dtype == EKV_INT32 && free_pages.shape[0] > kMost32)) {
        throw std::invalid_argument("int32 starts and new_head count at most 2^31 - 1 slots and free pages");
    }
    TableArgs a{};
    a.table = table.data;
    a.table_row = table.stride[0];
    a.table_col = table.stride[1];
    a.table64 = table.dtype == EKV_INT64;
    a.requests = table.shape[0];
    a.columns = table.shape[1];
    if (rows_p != nullptr) {
        a.rows = index_ref(need_vector(rows_p, batch, "rows"), 0);
    }
    a.lengths = index_ref(lengths, 0);
    a.added = index_ref(added, 0);
    a.free_pages = index_ref(free_pages, 0);
    a.free_head = index_ref(head, 0);
    a.slots = index_out(slots);
    a.starts = index_out(starts);
    a.new_lengths = index_out(new_lengths);
    a.new_head = index_out(new_head);
    a.capacity = slots.shape[0];
    const auto vector = [](const ekv_tensor& t) {
        return t.dtype == EKV_INT32 && t.stride[0] == 1 && reinterpret_cast<uintptr_t>(t.data) % 16 == 0;
    };
    a.vector = vector(slots);
    if (positions_p != nullptr) {
        const ekv_tensor& positions = need_vector(positions_p, a.capacity, "positions");
        a.positions = index_out(positions);
        a.has_positions = 1;
        a.vector = a.vector && vector(positions);
    }
    if (status_p != nullptr) {
        const ekv_tensor& status = need_vector(status_p, 1, "status");
        if (status.dtype != EKV_INT32) {
            throw std::invalid_argument("status must be int32");
        }
        a.status = static_cast<int32_t*>(status.data);
    }
    // Workgroups read the inputs while others write the outputs, and a repeated call reads them again.
    struct Array {
        Bytes bytes;
        const char* name;
    };
    const Array inputs[] = {{Bytes(&lengths), "lengths"}, {Bytes(&added), "added"}, {Bytes(rows_p), "rows"},
                            {Bytes(&free_pages), "free_pages"}, {Bytes(&head), "free_head"}};
    const Array outputs[] = {{Bytes(&new_lengths), "new_lengths"}, {Bytes(&new_head), "new_head"},
                             {Bytes(&starts), "starts"}, {Bytes(&slots), "slots"}, {Bytes(positions_p), "positions"},
                             {Bytes(status_p), "status"}};
    for (const Array& out : outputs) {
        const auto apart = [&](const Array& other) {
            if (out.bytes.meets(other.bytes)) {
                throw std::invalid_argument(std::string(out.name) + " must not share memory with " + other.name);
            }
        };
        for (const Array& in : inputs) {
            apart(in);
        }
        for (const Array* other = outputs; other != &out; ++other) {
            apart(*other);
        }
    }
    a.batch = batch;
    a.free_count = free_pages.shape[0];
    a.page_size = page_size;
    a.most_id = (std::numeric_limits<int64_t>::max() - (page_size - 1)) / page_size;
    a.page = FastDiv(static_cast<uint32_t>(page_size));
    const int64_t groups = std::min(std::max<int64_t>((a.capacity + kTile - 1) / kTile, 1), kMaxGroups);
    extend_tables_kernel<<<static_cast<uint32_t>(groups), kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
    check_hip(hipGetLastError(), "launch block tables");
    return 0;
}

}  // namespace
}  // namespace ekv

extern "C" int ekv_extend_block_tables(const ekv_tensor* block_tables, const ekv_tensor* rows,
                                       const ekv_tensor* lengths, const ekv_tensor* added,
                                       const ekv_tensor* free_pages, const ekv_tensor* free_head, int64_t page_size,
                                       const ekv_tensor* slots, const ekv_tensor* positions, const ekv_tensor* starts,
                                       const ekv_tensor* new_lengths, const ekv_tensor* new_head,
                                       const ekv_tensor* status, void* stream) {
    return ekv::guarded(-1, [&] {
        return ekv::extend_block_tables(block_tables, rows, lengths, added, free_pages, free_head, page_size, slots,
                                        positions, starts, new_lengths, new_head, status, stream);
    });
}
