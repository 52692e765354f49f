// The Top-K blocks of a request's context for each query token, by a score from 8-bit index keys (gfx950).
//
// With index query q_h of head h, held as codes (whole numbers of 8 bits) times a scale qs_h, and index key k_t of token
// t, codes times ks_t, the score of block j of block_size tokens for the query token at position p and a group of heads is
//   max over the group's heads h of  qs_h * max over t in block j, t <= p, of  ks_t * (q_h . k_t)
// with both products rounded to 32 bits. The sum q_h . k_t is a whole number below 2^24, so that neither the order of its
// terms nor its conversion rounds: scores have no freedom, and a selection is the same wherever it is made. Queries are
// rounded to codes here, as append.hip rounds keys.
//
// Two launches: scores of all blocks as ordered 32-bit keys into the workspace, then each (token, group)'s largest. Before
// them, for many query rows, one that makes the queries' codes.
#include "ekv_codes.h"
#include "ekv_device.h"
#include "ekv_memory.h"
#include "ekv_mfma.h"
#include "ekv_pool.h"
#include "ekv_vec.h"
#include "ekv_wave.h"

#include <algorithm>
#include <type_traits>

namespace ekv {
namespace {

constexpr int kThreads = 256, kWaves = 4;
// Keys of a wave's step: 8 KB of them at an index size of 128 or more.
constexpr int unit_of(int steps) { return steps == 4 ? 32 : 64; }

constexpr int kSegmentKeys = 4096;          // ordered keys of a workgroup's segment in LDS

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

struct BatchRows {
    IndexRef rows, lengths, query_starts;
    int32_t tokens, batch, requests;
    int32_t own_most;                       // tokens that a table row covers
};

struct ScoreArgs {
    const char* query;
    int64_t q_token, q_head;                // bytes
    int32_t f16;
    const char* keys;
    uint32_t page_stride, token_stride, pages;
    FastDiv page;
    const float* scales;
    int64_t scale_step;                     // elements
    const char* tables;
    int64_t table_row;                      // bytes
    uint32_t table_col;
    int32_t table64;
    BatchRows at;
    int32_t groups, share, dim;             // groups of share heads
    FastDiv group_div, share_div;
    FastDiv block;                          // tokens of a block
    int32_t block_units, sub_shift;         // steps of a block; or blocks of 2^sub_shift tokens, several a step (-1: not)
    uint32_t* scores;                       // [tokens, groups, score_row]
    int64_t score_row;
    char* codes;                            // queries as codes already, [tokens, groups, share] rows, and their scales;
    float* code_scales;                     // or NULL
    int32_t segment_blocks, segments;       // blocks of a segment; workgroups beside each other that share a tile's
    int32_t pairs;                          // (token, group) pairs of a tile of rows
    int32_t row_tiles;                      // tiles of a batch row with one query token
    int32_t tiles;
};

// Scores in the order of whole numbers: 0 for a block without a token that is seen, kForced for one that is always taken,
// which no score reaches. What passes the largest or the lowest number counts as that one.
constexpr uint32_t kForced = 0xff800000u;

// The score of what is not seen: NaN, of no account beside another in a maximum. (-infinity is a score: that of products
// that pass the lowest number.) The compiler is not to know it: it would make two maxima of three numbers again.
__device__ __forceinline__ float no_score() {
    uint32_t bits = 0x7fc00000u;
    asm("" : "+v"(bits));
    return __uint_as_float(bits);
}

__device__ __forceinline__ uint32_t ordered(float score) {
    const float most = 3.4028235e38f, held = __builtin_amdgcn_fmed3f(score, -most, most);
    const uint32_t bits = __float_as_uint(held + 0.0f);                            // -0 counts as 0
    const uint32_t key = bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
    return score == score ? key : 0u;
}

// The score of a key: infinity of kForced, NaN of 0.
__device__ __forceinline__ float score_of(uint32_t key) {
    return __uint_as_float(key ^ (~static_cast<uint32_t>(static_cast<int32_t>(key) >> 31) | 0x80000000u));
}

__device__ __forceinline__ int32_t clamped(int64_t v, int64_t low, int64_t high) {
    return static_cast<int32_t>(v < low ? low : (v > high ? high : v));
}

__device__ __forceinline__ int32_t first_token(const BatchRows& a, int32_t b) {
    return a.query_starts.data != nullptr ? clamped(a.query_starts.fetch(b), 0, a.tokens) : b;
}

// A batch row's tokens: query tokens first .. first + count - 1 at positions `position` ..; tokens 0 .. seen - 1 can be seen.
struct BatchRow {
    int32_t first, count, position, seen, request;
};

__device__ __forceinline__ BatchRow batch_row(const BatchRows& a, int32_t b) {
    BatchRow r;
    r.first = first_token(a, b);
    r.count = a.query_starts.data != nullptr ? max(first_token(a, b + 1) - r.first, 0) : 1;
    const int64_t length = a.lengths.fetch(b), request = a.rows.data != nullptr ? a.rows.fetch(b) : b;
    const bool good = request >= 0 && request < a.requests;
    r.request = good ? static_cast<int32_t>(request) : 0;
    r.seen = good ? clamped(length, 0, a.own_most) : 0;
    r.position = clamped(length, -1, 0x7ffffffe) - r.count;
    return r;
}

// The last batch row whose value is not above `wanted` (-1: none), where values do not decrease from row to row: 64 of them
// are looked at together, so that a call's first reads are two at most, one after the other, for 4096 rows. All lanes of
// a wave call it, with the same `wanted`.
template <typename Value>
__device__ __forceinline__ int32_t last_row_not_above(int32_t batch, int32_t wanted, Value&& value) {
    const int32_t lane = threadIdx.x & 63;
    int32_t low = 0, rows = batch;
    while (rows > 0) {
        const int32_t step = (rows + 63) >> 6, at = lane * step;
        const int32_t below = __popcll(__ballot(at < rows && value(low + min(at, rows - 1)) <= wanted));
        if (below == 0) {
            return low - 1;
        }
        // Row low + (below - 1) * step is not above it, the next of those looked at is.
        const int32_t begin = (below - 1) * step;
        if (step == 1) {
            return low + begin;
        }
        rows = min(step, rows - begin);
        low += begin;
    }
    return -1;
}

// The batch row whose query tokens hold `token` (a wave's), or -1.
__device__ __forceinline__ int32_t row_of_token(const BatchRows& a, int32_t token) {
    if (a.query_starts.data == nullptr) {
        return token < a.batch ? token : -1;
    }
    const int32_t b = last_row_not_above(a.batch, token, [&](int32_t row) { return first_token(a, row); });
    return b >= 0 && token < first_token(a, b + 1) ? b : -1;
}

__device__ __align__(256) const uint32_t no_key[64] = {};

__device__ __forceinline__ float over_quads_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Eight elements of an index query as codes, by the lanes that have its row (kSteps * 8 of them): all of a wave call it.
template <int kSteps>
__device__ __forceinline__ float query_codes(const ScoreArgs& a, bool live, int64_t token, int32_t head, int piece,
                                             uint32_t (&words)[2]) {
    float x[8] = {};
    float most = 0;
    if (live && piece * 8 < a.dim) {
        const u32x4 given = load_global<u32x4>(a.query + token * a.q_token + head * a.q_head + piece * 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint16_t bits = static_cast<uint16_t>(given[j >> 1] >> (16 * (j & 1)));
            x[j] = a.f16 != 0 ? F16::value(bits) : Bf16::value(bits);
            most = fmaxf(most, fabsf(x[j]));
        }
    }
#pragma unroll
    for (int step = 1; step < kSteps * 8; step *= 2) {
        most = fmaxf(most, __shfl_xor(most, step));
    }
    const float scale = code_scale(most);
    code_words(x, scale, words);
    return scale;
}

// All queries as codes, once, where many workgroups would each make the same ones: their making was 40 % of the
// instructions of a prompt's scores.
template <int kSteps>
__global__ __launch_bounds__(kThreads) void code_kernel(const ScoreArgs a) {
    constexpr int kRowThreads = kSteps * 8;
    const int64_t row = (int64_t{blockIdx.x} * kThreads + threadIdx.x) / kRowThreads;
    const int piece = threadIdx.x % kRowThreads;
    const bool live = row < int64_t{a.at.tokens} * a.groups * a.share;
    const int32_t heads = a.groups * a.share;
    const int64_t token = live ? row / heads : 0;
    uint32_t words[2];
    const float scale = query_codes<kSteps>(a, live, token, static_cast<int32_t>(row - token * heads), piece, words);
    if (live) {
        *reinterpret_cast<u32x2*>(a.codes + row * (kSteps * 64) + piece * 8) = u32x2{words[0], words[1]};
        if (piece == 0) {
            a.code_scales[row] = scale;
        }
    }
}

// Scores of a tile of rows (query heads of one batch row's tokens) against segments of its context. Keys down and rows
// across in 16x16x64 products, the tile's queries in registers, every wave with keys of its own: whole rows into registers
// while the keys before them are worked on, through LDS to the lanes that the products want. kShort: blocks of
// 2^sub_shift tokens, several a step.
//
// What bounds it: with few rows the reading. 5.2 million keys of 128 and their scales, 0.69 GB, of 128 requests of up to
// 65536 tokens take 130 us, 5.3 TB/s (lanes that read the products' way, 64 bytes of 16 rows, read each 128-byte line
// twice: 212). With many rows nothing alone: six pieces of up to 1024 tokens of 4 heads behind 16384 take 71 us, 0.77 *
// 10^15 operations a second, with the matrix pipes busy 15 % of the cycles, vector instructions (19 for 16 keys and 16
// rows) 36 %, and workgroups on the compute units two thirds of the time. Lists of tokens take longest for their
// bytes, a maximum in LDS for each key: 24 requests of up to 40000 tokens, 42 MB, 18 us.
template <int kSteps, int kTiles, bool kShort>
__global__ __launch_bounds__(kThreads, kSteps * kTiles > 16 ? 1 : 2) void score_kernel(const ScoreArgs a) {
    constexpr int kRowBytes = kSteps * 64, kPieces = kSteps * 4;
    constexpr int kUnit = unit_of(kSteps), kHalves = kUnit / 16;
    constexpr uint64_t kAll = kUnit == 64 ? ~uint64_t{0} : (uint64_t{1} << (kUnit & 63)) - 1;
    constexpr int kLanes = kPieces;                    // lanes that read a key's row
    constexpr int kAtOnce = 64 / kLanes;               // keys of one access
    constexpr int kLoads = kUnit / kAtOnce;
    static_assert(kTiles * 16 * kRowBytes <= kWaves * kUnit * kRowBytes, "codes fit where the keys will be");
    __shared__ __align__(16) char s_data[kWaves * kUnit * kRowBytes];      // the tile's codes, then each wave's keys
    __shared__ __align__(16) float s_scale[kTiles * 16 > kWaves * kUnit ? kTiles * 16 : kWaves * kUnit];
    extern __shared__ uint32_t s_score[];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups are dealt to the eight dies in turn, and a context's segments with them: long and short contexts, and the
    // early segments that all have, are everybody's.
    int32_t segment = blockIdx.x / a.tiles;
    const int32_t tile = (blockIdx.x + segment) % a.tiles;
    int32_t b, part;
    if (a.at.query_starts.data == nullptr) {
        b = tile / a.row_tiles, part = tile - b * a.row_tiles;
    } else {
        // Batch row b has tiles from starts[b] * groups / pairs + b on.
        const auto begin = [&](int32_t row) {
            return static_cast<int32_t>(int64_t{first_token(a.at, row)} * a.groups / a.pairs) + row;
        };
        b = __builtin_amdgcn_readfirstlane(last_row_not_above(a.at.batch, tile, begin));
        part = b >= 0 ? tile - begin(b) : -1;
    }
    if (b < 0 || b >= a.at.batch || part < 0) {
        return;
    }
    const BatchRow row = batch_row(a.at, b);
    const int32_t pair_begin = part * a.pairs, pair_count = min(row.count * a.groups - pair_begin, a.pairs);
    if (pair_count <= 0) {
        return;
    }
    // Of the tile's tokens: where the first and the last one's sight ends.
    const int32_t first_seen = min(row.position + static_cast<int32_t>(a.group_div.div(pair_begin)) + 1, row.seen);
    const int32_t last_seen =
        min(row.position + static_cast<int32_t>(a.group_div.div(pair_begin + pair_count - 1)) + 1, row.seen);
    if (last_seen <= 0 || segment * int64_t{a.segment_blocks} * a.block.divisor >= last_seen) {
        return;
    }

    i32x4 q[kTiles][kSteps];
    float q_scale[kTiles];
    int32_t sight[kTiles], pair_of[kTiles];        // of the lane's row of each 16; pair -1: no row
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
        const int32_t pair = a.share_div.div(m * 16 + col);
        pair_of[m] = pair < pair_count ? pair : -1;
        sight[m] = row.position + static_cast<int32_t>(a.group_div.div(pair_begin + max(pair_of[m], 0))) + 1;
    }
    if (a.codes != nullptr) {
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            const int r = m * 16 + col;
            const int64_t at = (int64_t{row.first} * a.groups + pair_begin) * a.share + r;
            const char* codes = pair_of[m] >= 0 ? a.codes + at * kRowBytes + quad * 16 : reinterpret_cast<const char*>(no_key);
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                q[m][c] = load_global<i32x4>(codes + (pair_of[m] >= 0 ? c * 64 : 0));
            }
            q_scale[m] = load_global<float>(pair_of[m] >= 0 ? reinterpret_cast<const char*>(a.code_scales + at)
                                                            : reinterpret_cast<const char*>(no_key));
        }
    } else {
        constexpr int kRowThreads = kSteps * 8;
        const int piece = tid % kRowThreads;
        for (int r = tid / kRowThreads; r < kTiles * 16; r += kThreads / kRowThreads) {
            const int32_t pair = a.share_div.div(r), all = pair_begin + pair, token = a.group_div.div(all);
            const int32_t head = (all - token * a.groups) * a.share + r - pair * a.share;
            uint32_t words[2];
            const float scale = query_codes<kSteps>(a, pair < pair_count, row.first + token, head, piece, words);
            const int at = r * kRowBytes + (((piece >> 1) ^ (r & (kPieces - 1))) << 4) + (piece & 1) * 8;
            *reinterpret_cast<u32x2*>(s_data + at) = u32x2{words[0], words[1]};
            if (piece == 0) {
                s_scale[r] = scale;
            }
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            const int r = m * 16 + col;
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                q[m][c] = *reinterpret_cast<const i32x4*>(s_data + r * kRowBytes +
                                                          (((c * 4 + quad) ^ (r & (kPieces - 1))) << 4));
            }
            q_scale[m] = s_scale[r];
        }
        lds_barrier();      // the keys come where the codes are
    }
    const char* const table = a.tables + row.request * a.table_row;
    const char* const nothing = reinterpret_cast<const char*>(no_key);
    const int32_t block_tokens = a.block.divisor, blocks = a.block.div(last_seen - 1) + 1;   // of the context

    for (; segment * int64_t{a.segment_blocks} < blocks; segment += a.segments) {
        const int32_t block_begin = segment * a.segment_blocks, held = min(a.segment_blocks, blocks - block_begin);
        for (int i = tid; i < pair_count * held; i += kThreads) {
            s_score[i] = 0;
        }
        lds_barrier();
        const int32_t begin = block_begin * block_tokens;
        // The context's last block may end early: every step begins at a token that somebody sees.
        const int32_t units = kShort
                                  ? (min(held << a.sub_shift, last_seen - begin) + kUnit - 1) / kUnit
                                  : (held - 1) * a.block_units +
                                        (min(block_tokens, last_seen - begin - (held - 1) * block_tokens) + kUnit - 1) / kUnit;
        const int32_t from = units * wave / kWaves, to = units * (wave + 1) / kWaves;

        // A wave's steps one after the other: kUnit tokens from `base` on, those before `end`.
        const int32_t span = kShort ? 0x7fffffff : block_tokens;      // tokens that steps go through in a run
        struct Step {
            int32_t left, start, offset, end;      // steps to come; first token of the block, and how far in it
            __device__ __forceinline__ int32_t base() const { return start + offset; }
        };
        const auto end_of = [&](int32_t start) { return last_seen - start > span ? start + span : last_seen; };
        const auto advance = [&](Step& s) {
            s.left -= 1;
            if (s.left <= 0) {
                s.end = 0;                         // nothing is read behind the last step
                return;
            }
            s.offset += kUnit;
            if (s.offset >= span) {
                s.start += span, s.offset = 0;
                s.end = end_of(s.start);
            }
        };
        // Page ids of a step: lane l's is that of its l-th key (an int64 id whose high word is not zero names no page).
        struct Ids {
            uint32_t low, high, inside;
        };
        const auto ids_of = [&](const Step& step) {
            const int32_t key = step.base() + lane;
            const bool good = lane < kUnit && key < step.end;
            const uint32_t page = a.page.div(key);
            const char* at = good ? table + uint64_t{page} * a.table_col : nothing;
            return Ids{load_global<uint32_t>(at), load_global<uint32_t>(at + (a.table64 != 0 ? 4 : 0)),
                       good ? key - page * a.page.divisor : ~0u};
        };
        // Rows of a step in registers: every access reads whole rows of kAtOnce keys, 16 bytes a lane. (With the lanes of
        // the matrix tiles it would read 64 bytes of each of 16 keys, and each 128-byte line twice.)
        struct Keys {
            i32x4 row[kLoads];
            float scale;                   // of key `lane`
            uint64_t seen;
        };
        const int my_piece = lane % kLanes * 16, my_key = lane / kLanes;
        const char* const from_piece = a.keys + (my_piece < a.dim ? my_piece : 0);     // the others meet codes of 0
        const auto fetch = [&](const Ids& e, Keys& keys) {
            const bool good = e.inside != ~0u && e.low >= 1 && e.low < a.pages && (a.table64 == 0 || e.high == 0);
            const char* scale_at = reinterpret_cast<const char*>(a.scales) +
                                   (uint64_t{e.low} * a.page.divisor + e.inside) * a.scale_step * 4;
            keys.scale = load_global<float>(good ? scale_at : nothing);
            keys.seen = __ballot(good);
            const uint64_t offset = uint64_t{e.low} * a.page_stride + uint64_t{e.inside} * a.token_stride;
            const uint32_t low = good ? static_cast<uint32_t>(offset) : ~0u;
            const uint32_t high = good ? static_cast<uint32_t>(offset >> 32) : ~0u;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t l = __shfl(low, i * kAtOnce + my_key), h = __shfl(high, i * kAtOnce + my_key);
                const char* at = from_piece + (uint64_t{h} << 32 | l);
                keys.row[i] = load_global<i32x4>(h != ~0u ? at : nothing);
            }
        };
        // Keys in LDS, their 16-byte pieces permuted by exclusive or so that 16 lanes with 16 keys and one piece meet every
        // bank once. Nobody but the wave reads them, and its accesses stay in order.
        char* const my_keys = s_data + wave * (kUnit * kRowBytes);
        float* const my_scales = s_scale + wave * kUnit;
        const auto swap_of = [](int key) {
            return kSteps == 1 ? (key >> 2) & 3 : (kSteps == 2 ? (key >> 1) & 7 : key & 15);
        };
        const auto put = [&](const Keys& keys) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int key = i * kAtOnce + my_key;
                *reinterpret_cast<i32x4*>(my_keys + key * kRowBytes + ((lane % kLanes ^ swap_of(key)) << 4)) = keys.row[i];
            }
            if (lane < kUnit) {
                my_scales[lane] = keys.scale;
            }
        };
        const float none = no_score();
        float best[kTiles];
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            best[m] = none;
        }
        const auto leave = [&](int m, float score, int32_t block) {
            if (pair_of[m] >= 0 && block < held) {
                atomicMax(&s_score[pair_of[m] * held + block], ordered(score * q_scale[m]));
            }
        };
        // The scores of the keys in LDS, 16 of them at a time; kRagged: some are not seen by all rows.
        const auto score = [&]<bool kRagged>(const Step& now, uint64_t seen, std::bool_constant<kRagged>) {
            const int32_t base = now.base();
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
            i32x4 k[kSteps];
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                k[c] = *reinterpret_cast<const i32x4*>(my_keys + (h * 16 + col) * kRowBytes +
                                                       (((c * 4 + quad) ^ swap_of(col)) << 4));
            }
            const f32x4 key_scale = *reinterpret_cast<const f32x4*>(my_scales + h * 16 + quad * 4);
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
                if (kRagged) {
                    __builtin_amdgcn_sched_barrier(0);     // masks of one tile at a time: scalar registers are few
                }
                i32x4 s = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < kSteps; ++c) {
                    s = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[c], q[m][c], s, 0, 0, 0);
                }
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[j] = static_cast<float>(s[j]) * key_scale[j];
                    if (kRagged) {
                        const int key = quad * 4 + j;
                        // Not &&, which became branches.
                        const bool there = (((seen >> (h * 16)) >> key & 1) != 0) & (key < sight[m] - base - h * 16);
                        x[j] = there ? x[j] : none;
                    }
                }
                if constexpr (!kShort) {
                    best[m] = fmaxf(fmaxf(best[m], x[0]), x[1]);
                    best[m] = fmaxf(fmaxf(best[m], x[2]), x[3]);
                } else {
                    const int32_t key = base - begin + h * 16 + quad * 4;      // from the segment's first
                    if (a.sub_shift == 0) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            leave(m, x[j], key + j);
                        }
                    } else if (a.sub_shift == 1) {
                        leave(m, fmaxf(x[0], x[1]), key >> 1);
                        leave(m, fmaxf(x[2], x[3]), (key >> 1) + 1);
                    } else {
                        leave(m, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), key >> a.sub_shift);
                    }
                }
            }
            }
        };
        const auto work = [&](const Step& now, uint64_t seen) {
            if (seen == kAll && now.base() + kUnit <= first_seen) {
                score(now, seen, std::false_type{});
            } else {
                rarely();
                score(now, seen, std::true_type{});
            }
            if (!kShort && (now.left == 1 || now.offset + kUnit >= span)) {
                const int32_t block = a.block.div(now.start - begin);
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
                    const float most = over_quads_max(best[m]);
                    if (quad == 0) {
                        leave(m, most, block);
                    }
                    best[m] = none;
                }
            }
        };
        if (from < to) {
            // Page ids are asked for two steps ahead, rows one.
            Step now;
            const int32_t block = kShort ? 0 : from / a.block_units;
            now.left = to - from;
            now.start = begin + (kShort ? 0 : block * block_tokens);
            now.offset = (from - (kShort ? 0 : block * a.block_units)) * kUnit;
            now.end = end_of(now.start);
            Step ahead = now;
            const Ids first = ids_of(ahead);
            advance(ahead);
            Ids ids = ids_of(ahead);
            advance(ahead);
            Keys keys;
            fetch(first, keys);
#pragma unroll 1
            for (; now.left > 0; advance(now)) {
                const Ids later = ids_of(ahead);
                advance(ahead);
                const uint64_t seen = keys.seen;
                put(keys);
                fetch(ids, keys);
                ids = later;
                work(now, seen);
            }
        }
        lds_barrier();
        for (int i = tid; i < pair_count * held; i += kThreads) {
            const int32_t pair = i / held, block = i - pair * held;
            a.scores[(int64_t{row.first} * a.groups + pair_begin + pair) * a.score_row + block_begin + block] = s_score[i];
        }
        lds_barrier();
    }
}

__device__ __forceinline__ uint32_t uniform_lane(uint32_t scanned) {
    return __builtin_amdgcn_readlane(scanned, 63);
}

// Keeps the compiler from making the masks of all of a wave's registers before it counts the first: it has scalar
// registers for few.
__device__ __forceinline__ void few_at_once(int r) {
    if (r % 8 == 7) {
        __builtin_amdgcn_sched_barrier(0);
    }
}

struct PickArgs {
    const uint32_t* scores;
    int64_t score_row;
    BatchRows at;
    FastDiv block, group_div;
    int32_t groups, chosen, first, last;
    int32_t* blocks;
    int64_t b_token, b_group, b_column;     // elements
};

// The blocks of a (token, group): those up to its newest, and the ones that are always taken.
struct Candidates {
    const uint32_t* scores;
    int32_t count, forced_below, forced_from;

    // Block j's key, given what is held for it.
    __device__ __forceinline__ uint32_t key_of(int32_t j, uint32_t k) const {
        k = j < count ? k : 0u;
        return k != 0 && (j < forced_below || j >= forced_from) ? kForced : k;
    }

    __device__ __forceinline__ uint32_t held(int32_t j) const {
        return load_global<uint32_t>(reinterpret_cast<const char*>(scores + max(min(j, count - 1), 0)));
    }

    // Whether some of blocks j .. j + 63 are always taken or past the end.
    __device__ __forceinline__ bool mixed(int32_t j) const {
        return j < forced_below || j + 63 >= forced_from || j + 63 >= count;
    }
};

__device__ __forceinline__ Candidates candidates_of(const PickArgs& a, int64_t pair) {
    const int32_t token = a.group_div.div(static_cast<uint32_t>(pair));
    const int32_t b = row_of_token(a.at, token);
    Candidates c{a.scores + pair * a.score_row, 0, a.first, 0};
    if (b >= 0) {
        const BatchRow row = batch_row(a.at, b);
        const int32_t position = row.position + (token - row.first);
        const int32_t seen = min(position + 1, row.seen);
        c.count = seen > 0 ? a.block.div(seen - 1) + 1 : 0;
        c.forced_from = position >= 0 ? static_cast<int32_t>(a.block.div(position)) + 1 - a.last : 0;
    }
    c.count = __builtin_amdgcn_readfirstlane(c.count);
    c.forced_from = __builtin_amdgcn_readfirstlane(c.forced_from);
    return c;
}

// A workgroup of kWaves waves a (token, group), or a wave each where kWaves is 1; wave w holds the w-th equal run of its
// blocks, 64 to a register. The K-th largest key bit by bit, by counting the keys that are not below a bound: that takes
// no order of the keys and no atomics, and stops as soon as exactly K are not below. Then the keys above the bound and the
// first of those equal to it, in order of their blocks. The bits that all keys share in front are skipped.
//
// What bounds it: the reads of the keys and the steps one after the other: kRegs comparisons and, between waves, a barrier
// a bit. 256 lists of up to 1024 blocks take 9.5 us, 4 lists of 64 3.5.
template <int kWaves, int kRegs>
__global__ __launch_bounds__(kWaves == 1 ? kThreads : kWaves * 64) void pick_kernel(const PickArgs a) {
    constexpr int kCells = kWaves == 1 ? 1 : kWaves;
    __shared__ uint32_t s_cells[2][2][kCells];
    const int lane = threadIdx.x & 63;
    const int in_group = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int wave = kWaves == 1 ? 0 : in_group;
    const int64_t pair = kWaves == 1 ? int64_t{blockIdx.x} * (kThreads / 64) + in_group : blockIdx.x;
    if (pair >= int64_t{a.at.tokens} * a.groups) {
        return;
    }
    const Candidates c = candidates_of(a, pair);
    const int32_t used = (c.count + kWaves * 64 - 1) / (kWaves * 64);     // registers
    const int32_t begin = wave * used * 64;
    uint32_t key[kRegs];
    uint32_t least = 0xffffffffu, most = 0;
#pragma unroll
    for (int r = 0; r < kRegs; ++r) {
        const int32_t j = begin + r * 64 + lane;
        key[r] = r < used ? c.key_of(j, c.held(j)) : 0u;
        // What is none, or always taken, says nothing of where the K-th largest lies.
        least = min(least, key[r] != 0 ? key[r] : 0xffffffffu);
        most = max(most, key[r] != kForced ? key[r] : 0u);
    }
    int parity = 0;
    // One number of each wave (the same in all its lanes), all of them to everybody.
    const auto share = [&](uint32_t first, uint32_t second, auto&& each) {
        if constexpr (kWaves > 1) {
            if (lane == 0) {
                s_cells[parity][0][wave] = first, s_cells[parity][1][wave] = second;
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                each(w, s_cells[parity][0][w], s_cells[parity][1][w]);
            }
            parity ^= 1;     // the next call's barrier stands between these reads and the writes after it
        } else {
            each(0, first, second);
        }
    };
    const auto not_below = [&](uint32_t bound) {
        uint32_t n = 0;
#pragma unroll
        for (int r = 0; r < kRegs; ++r) {
            n += __popcll(__ballot(key[r] >= bound));
            few_at_once(r);
        }
        int32_t all = 0;
        share(n, 0, [&](int, uint32_t x, uint32_t) { all += static_cast<int32_t>(x); });
        return all;
    };
    {
        const uint32_t low = ~uniform_lane(wave_scan<kMax>(~least)), high = uniform_lane(wave_scan<kMax>(most));
        least = 0xffffffffu, most = 0;
        share(low, high, [&](int, uint32_t x, uint32_t y) { least = min(least, x), most = max(most, y); });
    }
    // The K-th largest begins with the bits that the least and the largest share. With fewer than K keys the bound ends not
    // above the least, with K that are always taken not below the largest of the others: either way those are taken.
    const uint32_t differ = least ^ most;
    const int top = differ != 0 ? 31 - __builtin_clz(differ) : -1;
    uint32_t bound = top >= 31 ? 0u : (top < 0 ? least : least & ~((2u << top) - 1));
    bool exact = false;
    for (int bit = top; bit >= 0 && !exact; --bit) {
        const uint32_t tried = bound | (1u << bit);
        const int32_t n = not_below(tried);
        bound = n >= a.chosen ? tried : bound;
        exact = n == a.chosen;
    }
    const int32_t above = bound == 0xffffffffu ? 0 : not_below(bound + 1);
    int32_t equal = max(a.chosen - above, 0);                            // how many equal to the bound are taken
    const int32_t token = a.group_div.div(static_cast<uint32_t>(pair)), group = static_cast<int32_t>(pair) - token * a.groups;
    int32_t* const out = a.blocks + token * a.b_token + group * a.b_group;
    int32_t at = 0, taken_all = 0;
    if constexpr (kWaves > 1) {
        uint32_t mine_above = 0, mine_same = 0;
#pragma unroll
        for (int r = 0; r < kRegs; ++r) {
            mine_above += __popcll(__ballot(key[r] > bound));
            mine_same += __popcll(__ballot(bound != 0 && key[r] == bound));
            few_at_once(r);
        }
        int32_t same_before = 0, above_before = 0, same_all = 0;
        share(mine_above, mine_same, [&](int w, uint32_t x, uint32_t y) {
            above_before += w < wave ? x : 0, same_before += w < wave ? y : 0;
            same_all += y;
        });
        at = above_before + min(same_before, equal);
        taken_all = above + min(same_all, equal);
        equal -= min(same_before, equal);
    }
#pragma unroll
    for (int r = 0; r < kRegs; ++r) {
        const uint64_t same = __ballot(bound != 0 && key[r] == bound);
        const uint64_t mine = uint64_t{1} << lane;
        const bool take = key[r] > bound || ((same & mine) != 0 && __popcll(same & (mine - 1)) < equal);
        const uint64_t taken = __ballot(take);
        if (take) {
            out[(at + __popcll(taken & (mine - 1))) * a.b_column] = begin + r * 64 + lane;
        }
        at += __popcll(taken);
        equal -= min(equal, static_cast<int32_t>(__popcll(same)));
        few_at_once(r);
    }
    taken_all = kWaves == 1 ? at : taken_all;
    for (int32_t i = taken_all + (kWaves == 1 ? lane : static_cast<int32_t>(threadIdx.x)); i < a.chosen;
         i += kWaves == 1 ? 64 : kWaves * 64) {
        out[i * a.b_column] = -1;
    }
}

constexpr int kManyWaves = 16, kManyThreads = kManyWaves * 64;
constexpr int kDigit = 11, kBins = 1 << kDigit;
constexpr int kFew = 256;                     // keys that are compared with each other

// The same for many blocks. The range of the scores in 2047 equal parts, the keys counted in them, the part that holds
// the K-th largest; its keys, few as a rule, are compared with each other. (Parts of the range, not leading bits: those
// are the exponent, and most scores have one of few.) Where a part holds more than kFew, what is left is decided in digits
// of 11 bits of the key. kRegs: a lane's keys in registers; 0: any number of keys, read again each time.
//
// What bounds it: one compute unit has a list. 24 lists of 2048 out of up to 40000 tokens take 24 us: 6 for reading a
// list's 160 KB, 4 for counting, 4 for the few, 6 for counting those above and writing them, the rest in the steps between.
// (The K-th largest bit by bit from all keys took 94 us, by digits of 11 bits 49.)
template <int kRegs>
__global__ __launch_bounds__(kManyThreads) void pick_many_kernel(const PickArgs a) {
    __shared__ uint32_t s_bins[kBins];
    __shared__ __align__(16) uint32_t s_few[kFew];
    __shared__ uint32_t s_cells[2][kManyWaves];
    __shared__ uint32_t s_found[3];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t pair = blockIdx.x;
    const Candidates c = candidates_of(a, pair);
    const int32_t used = (c.count + kManyThreads - 1) / kManyThreads;      // a lane's keys
    const int32_t begin = wave * used * 64;
    uint32_t held[kRegs > 0 ? kRegs : 1];
    if constexpr (kRegs > 0) {
#pragma unroll
        for (int r = 0; r < kRegs; ++r) {
            held[r] = c.held(begin + min(r, used) * 64 + lane);
        }
#pragma unroll
        for (int r = 0; r < kRegs; ++r) {
            if (r >= used) {
                held[r] = 0;
            } else if (c.mixed(begin + r * 64)) {
                held[r] = c.key_of(begin + r * 64 + lane, held[r]);
            }
        }
    }
    // body(r, key) for each of a lane's keys, in order, and perhaps for keys of 0 behind them; whole waves take part.
    const auto for_keys = [&](auto&& body) {
        if constexpr (kRegs > 0) {
#pragma unroll
            for (int eight = 0; eight < kRegs; eight += 8) {
                if (eight < used) {
#pragma unroll
                    for (int r = eight; r < eight + 8; ++r) {
                        body(r, held[r]);
                        __builtin_amdgcn_sched_barrier(0);     // the masks of all would fill the scalar registers
                    }
                }
            }
        } else {
            for (int r = 0; r < used; ++r) {
                const int32_t j = begin + r * 64 + lane;
                body(r, c.key_of(j, c.held(j)));
            }
        }
    };
    // Values of each wave, the same in all its lanes, to all waves.
    const auto share = [&](uint32_t first, uint32_t second, auto&& each) {
        __syncthreads();
        if (lane == 0) {
            s_cells[0][wave] = first, s_cells[1][wave] = second;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kManyWaves; ++w) {
            each(w, s_cells[0][w], s_cells[1][w]);
        }
    };
    // The least and the largest of the keys that are neither none nor always taken: 0 - 1 and kForced - kForced are last.
    uint32_t least = 0xffffffffu, most = 0;
    for_keys([&](int, uint32_t key) {
        least = min(least, key - 1);
        most = max(most, key == kForced ? 0u : key);
    });
    {
        const uint32_t low = ~uniform_lane(wave_scan<kMax>(~least)), high = uniform_lane(wave_scan<kMax>(most));
        least = 0xffffffffu, most = 0;
        share(low, high, [&](int, uint32_t x, uint32_t y) { least = min(least, x), most = max(most, y); });
        least += 1;
    }
    uint32_t wanted = a.chosen;
    // Where, among the bins that place(key) counts keys in (-1: nowhere), the `wanted`-th largest is, of how many: false
    // if there are fewer. `wanted` becomes its place among those.
    const auto find = [&](auto&& place, uint32_t& bin, uint32_t& among) {
        __syncthreads();
        for (int i = tid; i < kBins; i += kManyThreads) {
            s_bins[i] = 0;
        }
        if (tid == 0) {
            s_found[0] = kBins;
        }
        __syncthreads();
        for_keys([&](int, uint32_t key) {
            const int at = place(key);
            if (at >= 0) {
                atomicAdd(&s_bins[at], 1u);
            }
        });
        __syncthreads();
        // From the largest down: two to a thread.
        const int top = kBins - 1 - 2 * tid;
        const uint32_t first = s_bins[top], second = s_bins[top - 1];
        const uint32_t sum = wave_scan<kAdd>(first + second);
        uint32_t before = sum - first - second;
        share(uniform_lane(sum), 0, [&](int w, uint32_t x, uint32_t) { before += w < wave ? x : 0; });
        if (before < wanted && wanted <= before + first + second) {
            const bool high = wanted <= before + first;
            s_found[0] = high ? top : top - 1;
            s_found[1] = high ? before : before + first;
            s_found[2] = high ? first : second;
        }
        __syncthreads();
        bin = s_found[0];
        if (bin == kBins) {
            return false;
        }
        wanted -= s_found[1];
        among = s_found[2];
        return true;
    };
    uint32_t from = 1, to = kForced, among = kFew + 1;       // the K-th largest is the wanted-th of `among` from .. to
    bool there = true;
    uint32_t bound = 0;                                      // all there are
    const float low = score_of(least), scale = (kBins - 2) / (score_of(most) - low);
    if (least < most && scale > 0 && scale < INFINITY) {
        // Parts 1 .. kBins - 1.
        const auto part = [&](uint32_t key) {
            return static_cast<int>(fminf(fmaf(score_of(key) - low, scale, 1.0f), kBins - 1));
        };
        uint32_t bin = 0;
        there = find([&](uint32_t key) { return key != 0 ? part(key) : -1; }, bin, among);
        if (there && among <= kFew) {
            // Each of them to a thread, which counts the larger ones.
            if (tid < kFew) {
                s_few[tid] = 0;
            }
            __syncthreads();
            if (tid == 0) {
                s_found[0] = 0;
            }
            __syncthreads();
            for_keys([&](int, uint32_t key) {
                if (key != 0 && part(key) == static_cast<int>(bin)) {
                    s_few[atomicAdd(&s_found[0], 1u)] = key;
                }
            });
            __syncthreads();
            if (tid < among) {
                const uint32_t mine = s_few[tid];
                uint32_t larger = 0, alike = 0;
                for (uint32_t i = 0; i < among; i += 4) {
                    const u32x4 some = *reinterpret_cast<const u32x4*>(s_few + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        larger += some[e] > mine, alike += some[e] == mine;
                    }
                }
                if (larger < wanted && wanted <= larger + alike) {
                    s_found[1] = mine, s_found[2] = larger;
                }
            }
            __syncthreads();
            bound = s_found[1];
            wanted -= s_found[2];
        }
        if (there && among > kFew) {
            // Its first and last key, by trying 64 keys at a time. Not those below the least: the keys of no score, NaN as
            // numbers, are among them, and parts do not increase from them on.
            const auto first_of = [&](int wanted_part) {
                uint32_t below = least - 1, above = kForced + 1;         // the first lies above `below`, not above `above`
                while (above - below > 1) {
                    const uint32_t step = (above - below + 63) / 64, at = below + min((lane + 1) * step, above - below);
                    const bool reached = at > kForced || part(at) >= wanted_part;
                    const int which = __builtin_ctzll(__ballot(reached));
                    above = below + min((which + 1) * step, above - below);
                    below += which * step;
                }
                return above;
            };
            from = first_of(bin), to = first_of(bin + 1) - 1;
        }
    }
    if (there && among > kFew) {
        const uint32_t differ = from ^ to;
        int bits = differ != 0 ? 32 - __builtin_clz(differ) : 0;
        bound = bits >= 32 ? 0u : (from >> bits) << bits;
        while (there && bits > 0) {
            const int digit = min(bits, kDigit), shift = bits - digit;
            uint32_t bin = 0;
            there = find(
                [&](uint32_t key) {
                    const bool mine = key >= from && key <= to && (bits >= 32 || (key ^ bound) >> bits == 0);
                    return mine ? static_cast<int>((key >> shift) & ((1u << digit) - 1)) : -1;
                },
                bin, among);
            bound |= bin << shift;
            bits = shift;
        }
        bound = there ? bound : 0u;
    }
    const int32_t equal = static_cast<int32_t>(wanted);      // how many equal to the bound are taken
    const int32_t token = a.group_div.div(static_cast<uint32_t>(pair)), group = static_cast<int32_t>(pair) - token * a.groups;
    int32_t* const out = a.blocks + token * a.b_token + group * a.b_group;
    uint32_t above = 0, same = 0;
    for_keys([&](int, uint32_t key) {
        above += key > bound;
        same += bound != 0 && key == bound;
    });
    above = uniform_lane(wave_scan<kAdd>(above)), same = uniform_lane(wave_scan<kAdd>(same));
    int32_t at = 0, same_before = 0, above_all = 0, same_all = 0;
    share(above, same, [&](int w, uint32_t x, uint32_t y) {
        at += w < wave ? x : 0, same_before += w < wave ? y : 0;
        above_all += x, same_all += y;
    });
    at += min(same_before, equal);
    int32_t left = max(equal - same_before, 0);              // of those equal to the bound, for this wave and later ones
    const uint64_t mine = uint64_t{1} << lane;
    // Never behind the list, not even where somebody else writes to the workspace and keys read again are others.
    const auto leave = [&](int r, bool take) {
        const uint64_t taken = __ballot(take);
        const int32_t place = at + static_cast<int32_t>(lanes_below(taken));
        if (take && place < a.chosen) {
            out[place * a.b_column] = begin + r * 64 + lane;
        }
        at += __popcll(taken);
    };
    const uint32_t limit = bound != 0 ? bound : 1u;
    if (bound == 0 || same_all <= equal) {
        for_keys([&](int r, uint32_t key) { leave(r, key >= limit); });
    } else {
        for_keys([&](int r, uint32_t key) {
            const uint64_t equals = __ballot(key == limit);
            const bool take = key > limit || ((equals & mine) != 0 && static_cast<int32_t>(lanes_below(equals)) < left);
            leave(r, take);
            left = max(left - static_cast<int32_t>(__popcll(equals)), 0);
        });
    }
    for (int32_t i = above_all + min(same_all, equal) + tid; i < a.chosen; i += kManyThreads) {
        out[i * a.b_column] = -1;
    }
}

// ---------------------------------------------------------------- host

constexpr int64_t kMostTokens = 1 << 23, kMostBatch = 1 << 20, kMostGroups = 1024, kMostShare = 128,
                  kMostPairs = (1 << 22) - 1;      // a workgroup each, of 1024 threads: fewer than 2^32 threads

// What the workspace keeps for the codes of a selection's queries: 1 KB of codes and a scale for each of up to 16 heads.
constexpr int64_t kCodeRoom = 1024, kScaleRoom = 64;

struct Plan {
    int64_t score_row = 0;
    uint64_t codes = 0, scales = 0;      // places in the workspace, behind the scores
    uint64_t bytes = 0;
};

Plan plan_of(int64_t tokens, int64_t groups, int64_t columns, int64_t page_size, int64_t block_size) {
    if (tokens < 0 || tokens > kMostTokens || groups < 1 || groups > kMostGroups) {
        throw std::invalid_argument("from 0 to 2^23 query tokens and from 1 to 1024 groups");
    }
    constexpr int64_t kMost = (int64_t{1} << 30) - 1;
    if (page_size < 1 || page_size > kMost || columns < 0 || columns > kMost / page_size) {
        throw std::invalid_argument("block_tables rows may cover at most 2^30 - 1 tokens");
    }
    if (block_size < 1 || block_size > (int64_t{1} << 30)) {
        throw std::invalid_argument("block_size must be from 1 to 2^30");
    }
    if (tokens * groups > kMostPairs) {
        throw std::invalid_argument("more than 2^22 - 1 selections");
    }
    Plan p;
    p.score_row = std::max<int64_t>((columns * page_size + block_size - 1) / block_size, 1);
    const auto aligned = [](uint64_t bytes) { return (bytes + 255) / 256 * 256; };
    const uint64_t lists = static_cast<uint64_t>(tokens * groups);
    p.codes = aligned(lists * static_cast<uint64_t>(p.score_row) * 4);
    p.scales = p.codes + lists * kCodeRoom;
    p.bytes = aligned(p.scales + lists * kScaleRoom);
    return p;
}

template <int kSteps, bool kShort>
void launch_tiles(const ScoreArgs& a, int tiles16, uint32_t grid, uint32_t lds, hipStream_t stream) {
    switch (tiles16) {
        case 1: score_kernel<kSteps, 1, kShort><<<grid, kThreads, lds, stream>>>(a); break;
        case 2: score_kernel<kSteps, 2, kShort><<<grid, kThreads, lds, stream>>>(a); break;
        case 4: score_kernel<kSteps, 4, kShort><<<grid, kThreads, lds, stream>>>(a); break;
        default: score_kernel<kSteps, 8, kShort><<<grid, kThreads, lds, stream>>>(a); break;
    }
    check_hip(hipGetLastError(), "launch block scores");
}

template <int kSteps>
void launch_scores(const ScoreArgs& a, int tiles16, uint32_t grid, uint32_t lds, hipStream_t stream) {
    if (a.sub_shift >= 0) {
        launch_tiles<kSteps, true>(a, tiles16, grid, lds, stream);
    } else {
        launch_tiles<kSteps, false>(a, tiles16, grid, lds, stream);
    }
}

int select_blocks(const ekv_select_args& s, void* workspace, uint64_t workspace_bytes, void* stream) {
    const ekv_tensor& query = need_rows(s.index_query, "index_query");
    const int64_t tokens = query.shape[0], heads = query.shape[1], dim = query.shape[2];
    if (dim < 16 || dim > 256 || dim % 16 != 0) {
        throw std::invalid_argument("the index size must be a multiple of 16 from 16 to 256");
    }
    const ekv_tensor& blocks = need(s.blocks, "blocks");
    need_ndim(blocks, 3, "blocks");
    need_dim(blocks, 0, tokens, "blocks");
    need_data(blocks, "blocks");
    if (blocks.dtype != EKV_INT32) {
        throw std::invalid_argument("blocks must be int32");
    }
    need_distinct(blocks, "blocks");
    const int64_t groups = blocks.shape[1], chosen = blocks.shape[2];
    if (groups < 1 || groups > kMostGroups || heads < 1 || heads % groups != 0 || heads / groups > kMostShare) {
        throw std::invalid_argument("blocks must have a divisor of the index heads as groups, at most 1024 of at most "
                                    "128 heads");
    }
    if (chosen < 1 || chosen > (int64_t{1} << 30)) {
        throw std::invalid_argument("blocks must hold from 1 to 2^30 blocks a list");
    }
    if (s.first < 0 || s.last < 0 || s.first > chosen || s.last > chosen - s.first) {
        throw std::invalid_argument("first and last must not be negative, and not more together than a list holds");
    }
    const ekv_tensor& tables = need(s.block_tables, "block_tables");
    need_ndim(tables, 2, "block_tables");
    need_index(tables, "block_tables");
    need_data(tables, "block_tables");
    const Plan plan = plan_of(tokens, groups, tables.shape[1], s.page_size, s.block_size);
    const PlanePages p = plane_pages(s.planes, s.layer, dim, s.page_size, 1);
    ScoreArgs a{};
    const ekv_tensor& scales = need(s.scales, "scales");
    need_ndim(scales, 1, "scales");
    need_data(scales, "scales");
    if (scales.dtype != EKV_FLOAT32) {
        throw std::invalid_argument("scales must be float32");
    }
    if (scales.shape[0] < p.pages * s.page_size) {
        throw std::invalid_argument("scales must have an element for each of the pool's " +
                                    std::to_string(p.pages * s.page_size) + " tokens, got " +
                                    std::to_string(scales.shape[0]));
    }
    const ekv_tensor& lengths = need(s.lengths, "lengths");
    need_ndim(lengths, 1, "lengths");
    need_index(lengths, "lengths");
    need_data(lengths, "lengths");
    if (lengths.shape[0] > kMostBatch) {
        throw std::invalid_argument("more than 2^20 batch rows");
    }
    a.at.tokens = static_cast<int32_t>(tokens);
    a.at.batch = static_cast<int32_t>(lengths.shape[0]);
    a.at.lengths = index_ref(lengths, 0);
    if (s.rows != nullptr) {
        a.at.rows = index_ref(need_list(s.rows, a.at.batch, "rows"), 0);
    }
    if (s.max_query < 1) {
        throw std::invalid_argument("max_query must be positive");
    }
    if (s.query_starts != nullptr) {
        a.at.query_starts = index_ref(need_list(s.query_starts, a.at.batch + 1, "query_starts"), 0);
    } else if (tokens != a.at.batch) {
        throw std::invalid_argument("without query_starts every batch row has one query token: got " +
                                    std::to_string(tokens) + " for " + std::to_string(a.at.batch) + " rows");
    }
    const Extent out(&blocks);
    need_apart(out, "blocks", Extent(&query), "index_query");
    need_apart(out, "blocks", Extent(p, *s.planes, 0), "the layer's plane");
    need_apart(out, "blocks", Extent(&scales), "scales");
    need_apart(out, "blocks", Extent(&tables), "block_tables");
    need_apart(out, "blocks", Extent(&lengths), "lengths");
    need_apart(out, "blocks", Extent(s.rows), "rows");
    need_apart(out, "blocks", Extent(s.query_starts), "query_starts");
    if (tokens == 0) {
        return 0;          // no workspace either: a tensor of its 0 bytes has no address
    }
    if (workspace_bytes < plan.bytes) {
        throw std::invalid_argument("the selection needs " + std::to_string(plan.bytes) + " workspace bytes, got " +
                                    std::to_string(workspace_bytes));
    }
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0) {
        throw std::invalid_argument("the workspace must be a 256-byte aligned device buffer");
    }
    const Extent work(workspace, plan.bytes);
    need_apart(work, "the workspace", out, "blocks");
    need_apart(work, "the workspace", Extent(&query), "index_query");
    need_apart(work, "the workspace", Extent(p, *s.planes, 0), "the layer's plane");
    need_apart(work, "the workspace", Extent(&scales), "scales");
    need_apart(work, "the workspace", Extent(&tables), "block_tables");
    need_apart(work, "the workspace", Extent(&lengths), "lengths");
    need_apart(work, "the workspace", Extent(s.rows), "rows");
    need_apart(work, "the workspace", Extent(s.query_starts), "query_starts");
    a.query = static_cast<const char*>(query.data);
    a.q_token = query.stride[0] * 2, a.q_head = query.stride[1] * 2;
    a.f16 = query.dtype == EKV_FLOAT16;
    a.keys = p.at;
    a.page_stride = static_cast<uint32_t>(p.page_stride), a.token_stride = static_cast<uint32_t>(p.token_stride);
    a.pages = static_cast<uint32_t>(p.pages);
    a.page = FastDiv(static_cast<uint32_t>(s.page_size));
    a.scales = static_cast<const float*>(scales.data);
    a.scale_step = scales.stride[0];
    a.tables = static_cast<const char*>(tables.data);
    a.table_row = tables.stride[0] * itemsize(tables.dtype);
    a.table_col = column_step(tables, "block_tables");
    a.table64 = tables.dtype == EKV_INT64;
    a.at.requests = static_cast<int32_t>(std::min<int64_t>(tables.shape[0], 0x7fffffff));
    a.at.own_most = static_cast<int32_t>(tables.shape[1] * s.page_size);
    a.groups = static_cast<int32_t>(groups), a.share = static_cast<int32_t>(heads / groups);
    a.dim = static_cast<int32_t>(dim);
    a.group_div = FastDiv(static_cast<uint32_t>(a.groups)), a.share_div = FastDiv(static_cast<uint32_t>(a.share));
    a.block = FastDiv(static_cast<uint32_t>(s.block_size));
    a.scores = static_cast<uint32_t*>(workspace);
    a.score_row = plan.score_row;
    const int64_t most_rows = std::min(s.max_query, tokens) * heads;
    // Row tiles of 16, 32, 64 and 128: calls of 4 heads of 128 for 32 requests of up to 16384 tokens take, with 4 query
    // tokens each, 26, 27, 30 and 31 us, with 8 tokens 39, 30, 30 and 32, with 16 tokens 57, 44, 31 and 36, four pieces
    // of 1024 tokens behind 8192 87, 79, 53 and 44.
    int tiles16 = most_rows <= 16 ? 1 : (most_rows <= 32 ? 2 : (most_rows <= 64 ? 4 : 8));
    while (16 * tiles16 < a.share) {
        tiles16 *= 2;
    }
    const int unit = unit_of(dim <= 64 ? 1 : (dim <= 128 ? 2 : 4));
    a.block_units = static_cast<int32_t>((s.block_size + unit - 1) / unit);
    a.sub_shift = -1;
    for (int shift = 0; 1 << shift < unit; ++shift) {
        if (s.block_size == 1 << shift) {
            a.sub_shift = shift;
        }
    }
    a.pairs = 16 * tiles16 / a.share;
    a.row_tiles = (a.groups + a.pairs - 1) / a.pairs;
    // Not none where there are no batch rows and nothing is scored.
    a.tiles = std::max(static_cast<int32_t>(s.query_starts != nullptr ? tokens * groups / a.pairs + a.at.batch
                                                                      : tokens * a.row_tiles), 1);
    // Segments of 256 tokens, of 512 where those fill the card twice, and longer where the contexts make more workgroups
    // than fill it a few times over (one for long tiles, whose start costs most); as many blocks as there is room for keys.
    // By 256, 512, 1024, 2048 and 4096 tokens: one query token of 4 heads for 4 requests of 8192 tokens 10, 11, 13, 17 and
    // 25 us, for 32 of 16384 26, 22, 23, 24 and 30, of 8 heads for 128 of 65536 181, 143, 138, 141 and 145; six pieces
    // of 600 behind 16384 126, 89, 77, 75 and 72 (by this rule 67), four of 1024 behind 8192 77, 57, 50, 44 and 66.
    const int64_t capacity = std::max<int64_t>(a.at.own_most, 1);
    const int64_t workgroups = tiles16 < 4 ? 8192 : (tiles16 == 4 ? 2048 : 512);
    const int64_t least = a.tiles * capacity / 512 >= 512 ? 512 : 256;
    const int64_t wanted = std::min<int64_t>(std::max<int64_t>(a.tiles * capacity / workgroups, least), 4096);
    int64_t segment_blocks = std::max<int64_t>(wanted / s.block_size, 1);
    segment_blocks = std::min<int64_t>(segment_blocks, kSegmentKeys / a.pairs);
    if (a.sub_shift >= 0) {
        // Whole steps: as many tokens as kSegmentKeys / 128 pairs leave room for are one at least.
        const int64_t each = unit >> a.sub_shift;
        segment_blocks = std::max<int64_t>(segment_blocks / each, 1) * each;
    }
    a.segment_blocks = static_cast<int32_t>(segment_blocks);
    const int64_t segments = std::min<int64_t>((plan.score_row + segment_blocks - 1) / segment_blocks,
                                         std::max<int64_t>(65536 / a.tiles, 1));
    a.segments = static_cast<int32_t>(segments);
    const uint32_t lds = static_cast<uint32_t>(a.pairs * segment_blocks * 4);
    const auto on = static_cast<hipStream_t>(stream);
    // Codes made once, by a launch of its own, where the rows are many: four pieces of 256 tokens of 4 heads behind 8192
    // take 33 instead of 38 us, 32 requests' 16 tokens each behind 16384 31 instead of 33. With few rows there is no
    // difference: 128 requests of one token behind 32768 take 87 and 88, 32 requests of 4 tokens 27 and 27.
    const int steps = dim <= 64 ? 1 : (dim <= 128 ? 2 : 4);
    if (tiles16 >= 4 && int64_t{a.share} * steps * 64 <= kCodeRoom && a.at.batch > 0) {
        a.codes = static_cast<char*>(workspace) + plan.codes;
        a.code_scales = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.scales);
        const uint32_t grid = static_cast<uint32_t>((tokens * heads * steps * 8 + kThreads - 1) / kThreads);
        switch (steps) {
            case 1: code_kernel<1><<<grid, kThreads, 0, on>>>(a); break;
            case 2: code_kernel<2><<<grid, kThreads, 0, on>>>(a); break;
            default: code_kernel<4><<<grid, kThreads, 0, on>>>(a); break;
        }
        check_hip(hipGetLastError(), "launch index query codes");
    }
    if (a.at.batch > 0) {
        const uint32_t grid = static_cast<uint32_t>(a.tiles * segments);
        if (dim <= 64) {
            launch_scores<1>(a, tiles16, grid, lds, on);
        } else if (dim <= 128) {
            launch_scores<2>(a, tiles16, grid, lds, on);
        } else {
            launch_scores<4>(a, tiles16, grid, lds, on);
        }
    }
    PickArgs k{};
    k.scores = a.scores;
    k.score_row = a.score_row;
    k.at = a.at;
    k.block = a.block, k.group_div = a.group_div;
    k.groups = a.groups, k.chosen = static_cast<int32_t>(chosen);
    k.first = static_cast<int32_t>(s.first), k.last = static_cast<int32_t>(s.last);
    k.blocks = static_cast<int32_t*>(blocks.data);
    k.b_token = blocks.stride[0], k.b_group = blocks.stride[1], k.b_column = blocks.stride[2];
    const uint32_t pairs = static_cast<uint32_t>(tokens * groups), grid = (pairs + kThreads / 64 - 1) / (kThreads / 64);
    // By a wave, by four, by sixteen, the last with keys in registers or read again each time. 4096 lists of the 256
    // blocks of 16384 tokens, a whole call: 94 us by a wave and 110 by four (8 lists: 11 and 14); of 2048 blocks 132 by
    // four and 205 by sixteen (8 lists: 16 and 15); of 16384 tokens 367 with 16 registers, 413 with 64 (8 lists: 19 and
    // 21); 8 lists of 65536 tokens 43 with 64 registers and 95 without.
    if (plan.score_row <= 256) {
        pick_kernel<1, 4><<<grid, kThreads, 0, on>>>(k);
    } else if (plan.score_row <= 2048) {
        pick_kernel<4, 8><<<pairs, 256, 0, on>>>(k);
    } else if (plan.score_row <= 16384) {
        pick_many_kernel<16><<<pairs, kManyThreads, 0, on>>>(k);
    } else if (plan.score_row <= 65536) {
        pick_many_kernel<64><<<pairs, kManyThreads, 0, on>>>(k);
    } else {
        pick_many_kernel<0><<<pairs, kManyThreads, 0, on>>>(k);
    }
    check_hip(hipGetLastError(), "launch block selection");
    return 0;
}

}  // namespace
}  // namespace ekv

extern "C" uint64_t ekv_select_workspace_bytes(int64_t tokens, int64_t groups, int64_t columns, int64_t page_size,
                                               int64_t block_size) {
    return ekv::guarded(~uint64_t{0}, [&] { return ekv::plan_of(tokens, groups, columns, page_size, block_size).bytes; });
}

extern "C" int ekv_select_blocks(const ekv_select_args* args, void* workspace, uint64_t workspace_bytes, void* stream) {
    return ekv::guarded(-1, [&] {
        if (args == nullptr) {
            throw std::invalid_argument("args is required");
        }
        return ekv::select_blocks(*args, workspace, workspace_bytes, stream);
    });
}
