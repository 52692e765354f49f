// New tokens into the paged pool (gfx950): queries and keys rotated by their positions, K and V rows put where the slot
// map says; and the tokens' 8-bit index keys beside them.
//
// Rotation. Pair i of a head, elements (x_a, x_b), is turned by the angle position * frequency_i:
//   y_a = x_a cos - x_b sin,   y_b = x_b cos + x_a sin
// A frequency is held as turns a position, a fraction of one turn in 64 bits. position * turns in 64-bit integers drops
// the whole turns by itself and adds no error: an angle is off by the position times what its frequency is, 4e-7 at 2^30
// for frequencies that were numbers of 64 bits (an angle in 32-bit floats would be off by 0.06 at position 10^6), and no
// table of cosines has to be read. The nearest quarter turn is split off as an integer too, and sine and cosine of the
// rest, at most pi / 4, are their power series in 32 bits.
//
// Index keys: rows as whole numbers of 8 bits (ekv_codes.h).
#include "ekv_codes.h"
#include "ekv_memory.h"
#include "ekv_mfma.h"
#include "ekv_pool.h"
#include "ekv_vec.h"

#include <cmath>

namespace ekv {
namespace {

constexpr int kThreads = 256;
constexpr int kMostPairs = 128;       // of a head of 256 elements
constexpr int kMostTokens = 4;        // of a workgroup
constexpr int kBatch = 4;             // units of a thread whose reads are under way together

// Where a slot's row begins in a plane.
struct SlotRows {
    FastDiv page;
    int64_t page_size, page_stride, token_stride;
    int64_t slots;                    // slots zero_below .. slots - 1 name rows
    int64_t zero_below;

    // The row's offset in bytes, or -1.
    __device__ __forceinline__ int64_t offset(int64_t slot) const {
        if (slot < zero_below || slot >= slots) {
            return -1;
        }
        const int64_t p = slot < 0x7fffffff ? page.div(static_cast<uint32_t>(slot)) : slot / page_size;
        return p * page_stride + (slot - p * page_size) * token_stride;
    }
};

struct Rows {
    const char* data;
    int64_t token, head;              // bytes
};

struct AppendArgs {
    Rows query, key, value;
    char* out;
    int64_t o_token, o_head;
    char* plane;                      // K of the layer; V at + kv_stride
    int64_t kv_stride;
    SlotRows rows;
    IndexRef positions, slots;
    const uint64_t* turns;            // 2^64 parts of a turn a position, of each pair
    float magnitude;
    int32_t tokens, each;             // tokens in all, of a workgroup
    int32_t q_heads, kv_heads;        // 0: not given
    int32_t head_bytes, half;         // bytes of a head; pairs
    int32_t pieces, rotated;          // pieces of a head; those that hold rotated elements
    FastDiv token_units, head_units;  // units of a token, of a head
};

struct CosSin {
    float cos, sin;
};

__device__ __forceinline__ CosSin turned(uint64_t phase) {
    const uint64_t eighth = uint64_t{1} << 61;
    const uint32_t quarter = static_cast<uint32_t>((phase + eighth) >> 62);
    // An eighth of a turn is 2^61: the rest fits the upper 32 bits of four times it.
    const int32_t rest = static_cast<int32_t>(static_cast<int64_t>(phase << 2) >> 32);
    const float x = static_cast<float>(rest) * 3.6572952e-10f;     // pi 2^-33
    const float xx = x * x;
    // To x^11 and x^10: what is left out is below 2^-34 and 2^-33.
    float s = -2.5052108e-8f;
    s = fmaf(s, xx, 2.7557319e-6f);
    s = fmaf(s, xx, -1.9841270e-4f);
    s = fmaf(s, xx, 8.3333333e-3f);
    s = fmaf(s, xx, -1.6666667e-1f);
    s = fmaf(s * xx, x, x);
    float c = -2.7557319e-7f;
    c = fmaf(c, xx, 2.4801587e-5f);
    c = fmaf(c, xx, -1.3888889e-3f);
    c = fmaf(c, xx, 4.1666667e-2f);
    c = fmaf(c, xx, -0.5f);
    c = fmaf(c, xx, 1.0f);
    const float swapped_c = (quarter & 1) != 0 ? s : c, swapped_s = (quarter & 1) != 0 ? c : s;
    return CosSin{((quarter + 1) & 2) != 0 ? -swapped_c : swapped_c, (quarter & 2) != 0 ? -swapped_s : swapped_s};
}

// kWidth elements in one access.
template <int kWidth>
struct Piece {
    uint16_t e[kWidth];
};

template <int kWidth>
__device__ __forceinline__ Piece<kWidth> load_piece(const char* at) {
    return __builtin_bit_cast(Piece<kWidth>, *reinterpret_cast<const typename Vec<2 * kWidth>::type*>(at));
}

template <int kWidth>
__device__ __forceinline__ void store_piece(char* at, const Piece<kWidth>& p) {
    *reinterpret_cast<typename Vec<2 * kWidth>::type*>(at) = __builtin_bit_cast(typename Vec<2 * kWidth>::type, p);
}

// A unit is two pieces of a head: pieces i and i + rotated / 2, which hold each other's pairs, and behind them the pieces
// that are only copied, two by two; where neighbours are pairs, pieces 2 i and 2 i + 1.
//
// What bounds it: the rows from and to HBM, and for a decode step the chain position -> angle -> store. Sines and cosines
// are computed once a token for all heads and shared through LDS. 25 thousand tokens of 48 heads of 128, 0.62 GB read and
// written, take 122 us, 5.1 TB/s (129 when the first rows were asked for behind the angles); 128 tokens 4.0 us.
template <typename T, int kWidth, bool kNeighbours>
__global__ __launch_bounds__(kThreads) void append_kernel(const AppendArgs a) {
    __shared__ __align__(16) float s_cos[kMostTokens * kMostPairs], s_sin[kMostTokens * kMostPairs];
    __shared__ int64_t s_row[kMostTokens];      // the row's offset, or -1
    __shared__ int32_t s_live[kMostTokens];
    const int tid = threadIdx.x;
    const int32_t first = blockIdx.x * a.each, count = min(a.each, a.tokens - first);
    const int32_t units = count * a.token_units.divisor;

    // A unit's pieces, and where they go but for the token's row.
    struct Unit {
        Piece<kWidth> x, y;
        int32_t token, head, low, high;          // head: of all, query, key and value
    };
    const auto unit_of = [&](int32_t u) {
        Unit r;
        r.token = a.token_units.div(u);
        const int32_t of_token = u - r.token * a.token_units.divisor;
        r.head = a.head_units.div(of_token);
        const int32_t unit = of_token - r.head * a.head_units.divisor;
        if (kNeighbours) {
            r.low = 2 * unit, r.high = r.low + 1;
        } else {
            const int32_t halves = a.rotated >> 1;
            r.low = unit < halves ? unit : 2 * unit;
            r.high = unit < halves ? unit + halves : r.low + 1;
        }
        return r;
    };
    const auto read = [&](Unit& r) {
        const int64_t at = first + r.token;
        const int32_t kv = r.head - a.q_heads;
        const char* from = a.query.data + at * a.query.token + r.head * a.query.head;
        if (kv >= a.kv_heads) {
            from = a.value.data + at * a.value.token + (kv - a.kv_heads) * a.value.head;
        } else if (kv >= 0) {
            from = a.key.data + at * a.key.token + kv * a.key.head;
        }
        // Behind the last piece the first of the two again.
        r.x = load_piece<kWidth>(from + r.low * (2 * kWidth));
        r.y = load_piece<kWidth>(from + (r.high < a.pieces ? r.high : r.low) * (2 * kWidth));
    };
    const auto finish = [&](Unit& r) {
        const int32_t kv = r.head - a.q_heads;
        const bool turns = kv < a.kv_heads;
        char* to;
        if (kv < 0) {
            to = s_live[r.token] != 0 ? a.out + (first + r.token) * a.o_token + r.head * a.o_head : nullptr;
        } else {
            const int64_t row = s_row[r.token];
            to = row >= 0 ? a.plane + (turns ? 0 : a.kv_stride) + row + (turns ? kv : kv - a.kv_heads) * a.head_bytes
                          : nullptr;
        }
        if (kNeighbours) {
            if constexpr (kWidth > 1) {
                const auto turn = [&](Piece<kWidth>& p, int32_t piece) {
                    const int place = r.token * kMostPairs + piece * (kWidth / 2);
#pragma unroll
                    for (int j = 0; j < kWidth; j += 2) {
                        const float c = s_cos[place + j / 2], s = s_sin[place + j / 2];
                        const float m = T::value(p.e[j]), n = T::value(p.e[j + 1]);
                        const uint32_t packed = T::pack(m * c - n * s, n * c + m * s);
                        p.e[j] = static_cast<uint16_t>(packed), p.e[j + 1] = static_cast<uint16_t>(packed >> 16);
                    }
                };
                if (turns && r.low < a.rotated) {
                    turn(r.x, r.low);
                }
                if (turns && r.high < a.rotated) {
                    turn(r.y, r.high);
                }
            }
        } else if (turns && r.low < a.rotated >> 1) {
            const int place = r.token * kMostPairs + r.low * kWidth;
#pragma unroll
            for (int j = 0; j < kWidth; ++j) {
                const float c = s_cos[place + j], s = s_sin[place + j];
                const float m = T::value(r.x.e[j]), n = T::value(r.y.e[j]);
                const uint32_t packed = T::pack(m * c - n * s, n * c + m * s);
                r.x.e[j] = static_cast<uint16_t>(packed), r.y.e[j] = static_cast<uint16_t>(packed >> 16);
            }
        }
        if (to != nullptr) {
            store_piece<kWidth>(to + r.low * (2 * kWidth), r.x);
            if (r.high < a.pieces) {
                store_piece<kWidth>(to + r.high * (2 * kWidth), r.y);
            }
        }
    };

    // The first units' rows are on their way while positions are read and angles computed.
    Unit held[kBatch];
    const auto read_batch = [&](int32_t base) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (base + k * kThreads < units) {
                held[k] = unit_of(base + k * kThreads);
                read(held[k]);
            }
        }
    };
    // Positions before rows: a wait for what was asked for later would be for the rows as well.
    constexpr int kAngles = kMostTokens * kMostPairs / kThreads;
    int32_t token_of[kAngles], pair_of[kAngles];
    int64_t position[kAngles], mine = 0, slot = 0;
    uint64_t turn[kAngles];
#pragma unroll
    for (int k = 0; k < kAngles; ++k) {
        const int i = tid + k * kThreads;
        if (i < count * a.half) {
            token_of[k] = i / a.half, pair_of[k] = i - token_of[k] * a.half;
            position[k] = a.positions.fetch(first + token_of[k]);
            turn[k] = a.turns[pair_of[k]];
        }
    }
    if (tid < count) {
        mine = a.positions.fetch(first + tid);
        slot = a.kv_heads > 0 ? a.slots.fetch(first + tid) : -1;
    }
    read_batch(tid);
#pragma unroll
    for (int k = 0; k < kAngles; ++k) {
        if (tid + k * kThreads < count * a.half) {
            const CosSin cs = turned(static_cast<uint64_t>(position[k]) * turn[k]);
            s_cos[token_of[k] * kMostPairs + pair_of[k]] = cs.cos * a.magnitude;
            s_sin[token_of[k] * kMostPairs + pair_of[k]] = cs.sin * a.magnitude;
        }
    }
    if (tid < count) {
        s_live[tid] = mine >= 0;
        s_row[tid] = mine >= 0 && a.kv_heads > 0 ? a.rows.offset(slot) : -1;
    }
    lds_barrier();
    for (int32_t base = tid; base < units; base += kBatch * kThreads) {
        if (base != tid) {
            read_batch(base);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (base + k * kThreads < units) {
                finish(held[k]);
            }
        }
    }
}

struct IndexArgs {
    const char* key;
    int64_t token;                    // bytes
    char* plane;
    float* scales;
    int64_t scale_step;               // elements
    SlotRows rows;
    IndexRef slots;
    int32_t tokens, pieces;           // pieces of 8 elements of a key
};

// kLanes lanes a token, 8 elements each: a row's largest magnitude without LDS. What bounds it: a launch, at the sizes that
// there are: 128 tokens of 64 take 2.5 us, 50 thousand of 128, 19 MB read and written, 8.
template <typename T, int kLanes>
__global__ __launch_bounds__(kThreads) void index_kernel(const IndexArgs a) {
    const int64_t token = (int64_t{blockIdx.x} * kThreads + threadIdx.x) / kLanes;
    const int piece = threadIdx.x % kLanes;
    const bool there = token < a.tokens, live = there && piece < a.pieces;
    float x[8] = {};
    float most = 0;
    if (live) {
        const Piece<8> p = load_piece<8>(a.key + token * a.token + piece * 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = T::value(p.e[j]);
            most = fmaxf(most, fabsf(x[j]));
        }
    }
#pragma unroll
    for (int step = 1; step < kLanes; step *= 2) {
        most = fmaxf(most, __shfl_xor(most, step));
    }
    const float scale = code_scale(most);
    uint32_t words[2];
    code_words(x, scale, words);
    const int64_t slot = there ? a.slots.fetch(token) : -1, row = a.rows.offset(slot);
    if (!live || row < 0) {
        return;
    }
    *reinterpret_cast<u32x2*>(a.plane + row + piece * 8) = u32x2{words[0], words[1]};
    if (piece == 0) {
        a.scales[slot * a.scale_step] = scale;
    }
}

// ---------------------------------------------------------------- host

constexpr int64_t kMostCount = 1 << 24;      // tokens of a call: a launch has fewer than 2^32 threads

SlotRows slot_rows(const PlanePages& p, int64_t page_size, int64_t rows, bool token_rows, int64_t zero_below) {
    if (zero_below < 0) {
        throw std::invalid_argument("zero_below must not be negative");
    }
    SlotRows r;
    // Where a plane row is a token, a slot is its row: also the rows behind the last whole page.
    r.page_size = token_rows ? 1 : page_size;
    r.page = FastDiv(static_cast<uint32_t>(r.page_size));
    r.page_stride = token_rows ? p.token_stride : p.page_stride;
    r.token_stride = p.token_stride;
    r.slots = token_rows ? rows : p.pages * page_size;
    r.zero_below = zero_below;
    return r;
}

Rows rows_of(const ekv_tensor& t) {
    return Rows{static_cast<const char*>(t.data), t.stride[0] * 2, t.stride[1] * 2};
}

template <typename T, int kWidth>
void launch_append(const AppendArgs& a, bool neighbours, hipStream_t stream) {
    const dim3 grid((a.tokens + a.each - 1) / a.each);
    if (!neighbours) {
        append_kernel<T, kWidth, false><<<grid, kThreads, 0, stream>>>(a);
    } else if constexpr (kWidth > 1) {
        append_kernel<T, kWidth, true><<<grid, kThreads, 0, stream>>>(a);
    }
    check_hip(hipGetLastError(), "launch append_rotary");
}

template <typename T>
void launch_append_type(const AppendArgs& a, int width, bool neighbours, hipStream_t stream) {
    switch (width) {
        case 8: launch_append<T, 8>(a, neighbours, stream); break;
        case 4: launch_append<T, 4>(a, neighbours, stream); break;
        case 2: launch_append<T, 2>(a, neighbours, stream); break;
        default: launch_append<T, 1>(a, neighbours, stream); break;
    }
}

int append_rotary(const ekv_append_args& s, void* stream) {
    const bool queries = s.query != nullptr, keys = s.key != nullptr;
    if (queries != (s.output != nullptr)) {
        throw std::invalid_argument("query and output are given together");
    }
    if (keys != (s.value != nullptr) || keys != (s.planes != nullptr) || keys != (s.slots != nullptr)) {
        throw std::invalid_argument("key, value, planes and slots are given together");
    }
    if (!queries && !keys) {
        throw std::invalid_argument("query or key is required");
    }
    const ekv_tensor& lead = need_rows(queries ? s.query : s.key, queries ? "query" : "key");
    const int64_t tokens = lead.shape[0], dim = lead.shape[2];
    if (dim < 8 || dim > 256 || dim % 8 != 0) {
        throw std::invalid_argument("the head size must be a multiple of 8 from 8 to 256");
    }
    constexpr int64_t kMostHeads = 65535;
    if (tokens > kMostCount) {
        throw std::invalid_argument("more than 2^24 tokens");
    }
    const auto same = [&](const ekv_tensor* p, const char* name) -> const ekv_tensor& {
        const ekv_tensor& t = need_rows(p, name);
        need_dim(t, 0, tokens, name);
        need_dim(t, 2, dim, name);
        if (t.dtype != lead.dtype) {
            throw std::invalid_argument(std::string(name) + " must have the type of " + (queries ? "query" : "key"));
        }
        if (t.shape[1] < 1 || t.shape[1] > kMostHeads) {
            throw std::invalid_argument(std::string(name) + " must have from 1 to 65535 heads");
        }
        return t;
    };
    AppendArgs a{};
    a.tokens = static_cast<int32_t>(tokens);
    const ekv_tensor& positions = need_list(s.positions, tokens, "positions");
    a.positions = index_ref(positions, 0);
    const ekv_tensor& turns = need(s.turns, "turns");
    need_ndim(turns, 1, "turns");
    need_data(turns, "turns");
    if (turns.dtype != EKV_INT64 || (turns.shape[0] > 1 && turns.stride[0] != 1) ||
        reinterpret_cast<uintptr_t>(turns.data) % 8 != 0) {
        throw std::invalid_argument("turns must be dense int64");
    }
    if (turns.shape[0] < 1 || 2 * turns.shape[0] > dim) {
        throw std::invalid_argument("turns must hold from 1 to half the head size's pairs");
    }
    a.half = static_cast<int32_t>(turns.shape[0]);
    a.turns = static_cast<const uint64_t*>(turns.data);
    a.magnitude = static_cast<float>(s.magnitude);
    if (!std::isfinite(a.magnitude)) {
        throw std::invalid_argument("magnitude must be finite");
    }
    a.head_bytes = static_cast<int32_t>(dim * 2);
    if (queries) {
        const ekv_tensor& query = same(s.query, "query");
        const ekv_tensor& out = same(s.output, "output");
        need_dim(out, 1, query.shape[1], "output");
        a.q_heads = static_cast<int32_t>(query.shape[1]);
        a.query = rows_of(query);
        a.out = static_cast<char*>(out.data);
        a.o_token = out.stride[0] * 2, a.o_head = out.stride[1] * 2;
        need_distinct(out, "output");
        const Extent o(&out);
        if (!same_view(query, out)) {
            need_apart(o, "output", Extent(&query), "query, unless it is the query");
        }
        need_apart(o, "output", Extent(&positions), "positions");
        need_apart(o, "output", Extent(&turns), "turns");
    }
    if (keys) {
        const ekv_tensor& key = same(s.key, "key");
        const ekv_tensor& value = same(s.value, "value");
        need_dim(value, 1, key.shape[1], "value");
        const ekv_tensor& slots = need_list(s.slots, tokens, "slots");
        a.kv_heads = static_cast<int32_t>(key.shape[1]);
        a.key = rows_of(key), a.value = rows_of(value);
        a.slots = index_ref(slots, 0);
        const int64_t row = a.kv_heads * dim * 2;
        const PlanePages p = plane_pages(s.planes, s.layer, row, s.page_size, 2);
        need_distinct_rows(*s.planes);
        a.rows = slot_rows(p, s.page_size, s.planes->rows, s.planes->row_bytes == row, s.zero_below);
        a.plane = p.at;
        a.kv_stride = p.kv_stride;
        const Extent planes[2] = {Extent(p, *s.planes, 0), Extent(p, *s.planes, 1)};
        const auto apart = [&](const ekv_tensor* t, const char* name) {
            for (const Extent& plane : planes) {
                need_apart(Extent(t), name, plane, "the layer's planes");
            }
            if (queries && t != s.query && t != s.output) {
                need_apart(Extent(s.output), "output", Extent(t), name);
            }
        };
        apart(s.key, "key");
        apart(s.value, "value");
        apart(s.slots, "slots");
        apart(s.positions, "positions");
        apart(s.turns, "turns");
        if (queries) {
            apart(s.query, "query");
            apart(s.output, "output");
        }
        need_apart(planes[0], "the layer's K plane", planes[1], "its V plane");
    }
    if (tokens == 0) {
        return 0;
    }
    const bool neighbours = s.interleaved != 0;
    // The widest access that lets a piece's pairs be whole: half the rotated elements hold whole pieces, or, where
    // neighbours are pairs, all of them.
    const int width = pick_vector_width({neighbours ? 4 * a.half : 2 * a.half}) / 2;
    a.pieces = static_cast<int32_t>(dim / width);
    a.rotated = 2 * a.half / width;
    const int64_t head_units = (a.pieces + 1) / 2, units = head_units * (a.q_heads + 2 * int64_t{a.kv_heads});
    a.head_units = FastDiv(static_cast<uint32_t>(head_units));
    a.token_units = FastDiv(static_cast<uint32_t>(units));
    // A workgroup takes one token while there are few, so that more of them share the reads: eight prompts' 25 thousand
    // tokens of 48 heads take 122 us by four, 121 by two and 133 by one, 2549 of 20 heads of 80 7.5, 8.5 and 10.4.
    a.each = tokens <= 1024 ? 1 : kMostTokens;
    const auto on = static_cast<hipStream_t>(stream);
    if (lead.dtype == EKV_BFLOAT16) {
        launch_append_type<Bf16>(a, width, neighbours, on);
    } else {
        launch_append_type<F16>(a, width, neighbours, on);
    }
    return 0;
}

template <typename T>
void launch_index(const IndexArgs& a, hipStream_t stream) {
    int lanes = 2;
    while (lanes < a.pieces) {
        lanes *= 2;
    }
    const dim3 grid(static_cast<uint32_t>((int64_t{a.tokens} * lanes + kThreads - 1) / kThreads));
    switch (lanes) {
        case 2: index_kernel<T, 2><<<grid, kThreads, 0, stream>>>(a); break;
        case 4: index_kernel<T, 4><<<grid, kThreads, 0, stream>>>(a); break;
        case 8: index_kernel<T, 8><<<grid, kThreads, 0, stream>>>(a); break;
        case 16: index_kernel<T, 16><<<grid, kThreads, 0, stream>>>(a); break;
        default: index_kernel<T, 32><<<grid, kThreads, 0, stream>>>(a); break;
    }
    check_hip(hipGetLastError(), "launch append_index");
}

int append_index(const ekv_tensor* key_p, const ekv_planes* planes, int64_t layer, int64_t page_size,
                 const ekv_tensor* scales_p, const ekv_tensor* slots_p, int64_t zero_below, void* stream) {
    const ekv_tensor& key = need(key_p, "index_key");
    need_ndim(key, 2, "index_key");
    if (key.dtype != EKV_BFLOAT16 && key.dtype != EKV_FLOAT16) {
        throw std::invalid_argument("index_key must be bfloat16 or float16");
    }
    need_data(key, "index_key");
    const int64_t tokens = key.shape[0], dim = key.shape[1];
    if (dim < 16 || dim > 256 || dim % 16 != 0) {
        throw std::invalid_argument("the index size must be a multiple of 16 from 16 to 256");
    }
    if (tokens > kMostCount) {
        throw std::invalid_argument("more than 2^24 tokens");
    }
    if (key.stride[1] != 1) {
        throw std::invalid_argument("index_key must be dense in its last dimension");
    }
    if (tokens > 0) {
        need_aligned(reinterpret_cast<int64_t>(key.data), "index_key address");
        need_aligned(tokens > 1 ? key.stride[0] * 2 : 0, "index_key token stride");
    }
    const ekv_tensor& slots = need_list(slots_p, tokens, "slots");
    const PlanePages p = plane_pages(planes, layer, dim, page_size, 1);
    IndexArgs a{};
    a.rows = slot_rows(p, page_size, planes->rows, planes->row_bytes == dim, zero_below);
    const ekv_tensor& scales = need(scales_p, "scales");
    need_ndim(scales, 1, "scales");
    need_data(scales, "scales");
    if (scales.dtype != EKV_FLOAT32) {
        throw std::invalid_argument("scales must be float32");
    }
    if (scales.shape[0] < a.rows.slots) {
        throw std::invalid_argument("scales must have an element for each of the pool's " +
                                    std::to_string(a.rows.slots) + " slots, got " + std::to_string(scales.shape[0]));
    }
    need_distinct(scales, "scales");
    need_distinct_rows(*planes);
    const Extent plane(p, *planes, 0), scale_extent(&scales);
    need_apart(Extent(&key), "index_key", plane, "the layer's plane");
    need_apart(Extent(&slots), "slots", plane, "the layer's plane");
    need_apart(scale_extent, "scales", plane, "the layer's plane");
    need_apart(scale_extent, "scales", Extent(&key), "index_key");
    need_apart(scale_extent, "scales", Extent(&slots), "slots");
    if (tokens == 0) {
        return 0;
    }
    a.key = static_cast<const char*>(key.data);
    a.token = key.stride[0] * 2;
    a.plane = p.at;
    a.scales = static_cast<float*>(scales.data);
    a.scale_step = scales.stride[0];
    a.slots = index_ref(slots, 0);
    a.tokens = static_cast<int32_t>(tokens);
    a.pieces = static_cast<int32_t>(dim / 8);
    const auto on = static_cast<hipStream_t>(stream);
    if (key.dtype == EKV_BFLOAT16) {
        launch_index<Bf16>(a, on);
    } else {
        launch_index<F16>(a, on);
    }
    return 0;
}

}  // namespace
}  // namespace ekv

extern "C" int ekv_append_rotary(const ekv_append_args* args, void* stream) {
    return ekv::guarded(-1, [&] {
        if (args == nullptr) {
            throw std::invalid_argument("args is required");
        }
        return ekv::append_rotary(*args, stream);
    });
}

extern "C" int ekv_append_index(const ekv_tensor* index_key, const ekv_planes* planes, int64_t layer, int64_t page_size,
                                const ekv_tensor* scales, const ekv_tensor* slots, int64_t zero_below, void* stream) {
    return ekv::guarded(-1, [&] {
        return ekv::append_index(index_key, planes, layer, page_size, scales, slots, zero_below, stream);
    });
}
