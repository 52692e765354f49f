// The Top-K blocks of a request's context for each query token, by a score from 8-bit index keys (gfx950).
//
// With index query q_h of head h, held as codes (whole numbers of 8 bits) times a scale qs_h, and index key k_t of token
// t, codes times ks_t, the score of block j of block_size tokens for the query token at position p and a group of heads is
//   max over the group's heads h of  qs_h * max over t in block j, t <= p, of  ks_t * (q_h . k_t)
// with both products rounded to 32 bits. The sum q_h . k_t is a whole number below 2^24, so that neither the order of its
// terms nor its conversion rounds: scores have no freedom, and a selection is the same wherever it is made. Queries are
// rounded to codes here, as append.hip rounds keys.
//
// Two launches: scores of all blocks as ordered 32-bit keys into the workspace, then each (token, group)'s largest.
#include "ekv_mfma.h"
#include "ekv_pool.h"
#include "ekv_vec.h"
#include "ekv_wave.h"

#include <algorithm>

namespace ekv {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kUnit = 32;                   // keys of a wave's step
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
    int32_t block_units, sub_shift;         // steps of a block; or blocks of 2^sub_shift < kUnit tokens (-1: not)
    uint32_t* scores;                       // [tokens, groups, score_row]
    int64_t score_row;
    int32_t segment_blocks, segments;       // blocks of a segment; workgroups beside each other that share a tile's
    int32_t pairs;                          // (token, group) pairs of a tile of rows
    int32_t row_tiles;                      // tiles of a batch row with one query token
    int32_t tiles;
};

// Scores in the order of whole numbers, 0 for a block without a token that is seen.
__device__ __forceinline__ uint32_t ordered(float score) {
    const uint32_t bits = __float_as_uint(score + 0.0f);     // -0 counts as 0
    const uint32_t key = bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
    return score > -INFINITY ? key : 0u;
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

// The batch row whose query tokens hold `token`, or -1.
__device__ __forceinline__ int32_t row_of_token(const BatchRows& a, int32_t token) {
    if (a.query_starts.data == nullptr) {
        return token < a.batch ? token : -1;
    }
    int32_t low = 0, high = a.batch;
    while (high - low > 1) {
        const int32_t mid = (low + high) >> 1;
        if (first_token(a, mid) <= token) {
            low = mid;
        } else {
            high = mid;
        }
    }
    return a.batch > 0 && first_token(a, low) <= token && token < first_token(a, low + 1) ? low : -1;
}

__device__ __align__(256) const uint32_t no_key[64] = {};

__device__ __forceinline__ float over_quads_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Scores of a tile of rows (query heads of one batch row's tokens) against segments of its context. Keys down and rows
// across in 16x16x64 products, every wave with keys of its own straight from memory, the tile's queries in its registers.
template <int kSteps, int kTiles>
__global__ __launch_bounds__(kThreads) void score_kernel(const ScoreArgs a) {
    constexpr int kRowBytes = kSteps * 64, kPieces = kSteps * 4;
    __shared__ __align__(16) char s_codes[kTiles * 16 * kRowBytes];
    __shared__ float s_scale[kTiles * 16];
    extern __shared__ uint32_t s_score[];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups are dealt to the eight dies in turn: those of one segment meet behind one L2.
    int32_t tile, segment;
    if (a.segments % 8 == 0) {
        const int32_t each = blockIdx.x >> 3;
        tile = each % a.tiles, segment = (each / a.tiles) * 8 + (blockIdx.x & 7);
    } else {
        tile = blockIdx.x % a.tiles, segment = blockIdx.x / a.tiles;
    }
    int32_t b, part;
    if (a.at.query_starts.data == nullptr) {
        b = tile / a.row_tiles, part = tile - b * a.row_tiles;
    } else {
        // Batch row b has tiles from starts[b] * groups / pairs + b on.
        const auto begin = [&](int32_t row) {
            return static_cast<int32_t>(int64_t{first_token(a.at, row)} * a.groups / a.pairs) + row;
        };
        int32_t low = 0, high = a.at.batch;
        while (high - low > 1) {
            const int32_t mid = (low + high) >> 1;
            if (begin(mid) <= tile) {
                low = mid;
            } else {
                high = mid;
            }
        }
        b = low, part = tile - begin(low);
    }
    if (b >= a.at.batch || part < 0) {
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

    // Queries as codes.
    {
        constexpr int kLanes = kSteps * 8;
        const int piece = tid % kLanes;
        for (int r = tid / kLanes; r < kTiles * 16; r += kThreads / kLanes) {
            const int32_t pair = a.share_div.div(r), inside = r - pair * a.share;
            float x[8] = {};
            float most = 0;
            if (pair < pair_count && piece * 8 < a.dim) {
                const int32_t all = pair_begin + pair, token = a.group_div.div(all);
                const int32_t head = (all - token * a.groups) * a.share + inside;
                const u32x4 words = *reinterpret_cast<const u32x4*>(
                    a.query + int64_t{row.first + token} * a.q_token + head * a.q_head + piece * 16);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint16_t bits = static_cast<uint16_t>(words[j >> 1] >> (16 * (j & 1)));
                    x[j] = a.f16 != 0 ? F16::value(bits) : Bf16::value(bits);
                    most = fmaxf(most, fabsf(x[j]));
                }
            }
#pragma unroll
            for (int step = 1; step < kLanes; step *= 2) {
                most = fmaxf(most, __shfl_xor(most, step));
            }
            const float scale = most / 127.0f, divisor = scale > 0 ? scale : 1.0f;
            u32x2 words = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int32_t code = static_cast<int32_t>(rintf(x[j] / divisor));
                words[j >> 2] |= (static_cast<uint32_t>(code) & 0xffu) << (8 * (j & 3));
            }
            const int at = r * kRowBytes + (((piece >> 1) ^ (r & (kPieces - 1))) << 4) + (piece & 1) * 8;
            *reinterpret_cast<u32x2*>(s_codes + at) = words;
            if (piece == 0) {
                s_scale[r] = scale;
            }
        }
    }
    __syncthreads();
    i32x4 q[kTiles][kSteps];
    float q_scale[kTiles];
    int32_t sight[kTiles], pair_of[kTiles];        // of the lane's row of each 16; pair -1: no row
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
        const int r = m * 16 + col;
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            q[m][c] = *reinterpret_cast<const i32x4*>(s_codes + r * kRowBytes + (((c * 4 + quad) ^ (r & (kPieces - 1))) << 4));
        }
        q_scale[m] = s_scale[r];
        const int32_t pair = a.share_div.div(r);
        pair_of[m] = pair < pair_count ? pair : -1;
        sight[m] = row.position + static_cast<int32_t>(a.group_div.div(pair_begin + max(pair_of[m], 0))) + 1;
    }
    const char* const table = a.tables + row.request * a.table_row;
    const char* const nothing = reinterpret_cast<const char*>(no_key);
    const int32_t block_tokens = a.block.divisor, blocks = a.block.div(last_seen - 1) + 1;   // of the context

    for (; segment * int64_t{a.segment_blocks} < blocks; segment += a.segments) {
        const int32_t block_begin = segment * a.segment_blocks, held = min(a.segment_blocks, blocks - block_begin);
        for (int i = tid; i < pair_count * held; i += kThreads) {
            s_score[i] = 0;
        }
        __syncthreads();
        const int32_t begin = block_begin * block_tokens;
        // The context's last block may end early: every step begins at a token that somebody sees.
        const int32_t units = a.sub_shift >= 0
                                  ? (min(held << a.sub_shift, last_seen - begin) + kUnit - 1) / kUnit
                                  : (held - 1) * a.block_units +
                                        (min(block_tokens, last_seen - begin - (held - 1) * block_tokens) + kUnit - 1) / kUnit;
        const int32_t from = units * wave / kWaves, to = units * (wave + 1) / kWaves;

        // First position of a step, and where its block's tokens end.
        const auto place = [&](int32_t u, int32_t& base, int32_t& end) {
            if (a.sub_shift >= 0) {
                base = begin + u * kUnit;
                end = min(row.seen, last_seen);
            } else {
                const int32_t block = u / a.block_units;
                base = begin + block * block_tokens + (u - block * a.block_units) * kUnit;
                end = min(begin + (block + 1) * block_tokens, last_seen);
            }
        };
        struct Ids {
            uint32_t low[2], high[2];
        };
        const auto ids_of = [&](int32_t u) {
            Ids e;
            int32_t base, end;
            place(min(u, units - 1), base, end);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int32_t key = base + h * 16 + col;
                const char* at = key < end ? table + uint64_t{a.page.div(key)} * a.table_col : nothing;
                e.low[h] = *reinterpret_cast<const uint32_t*>(at);
                e.high[h] = *reinterpret_cast<const uint32_t*>(at + (a.table64 != 0 ? 4 : 0));
            }
            return e;
        };
        i32x4 k[2][kSteps];
        float scale[2];
        uint32_t seen = 0;
        const auto fetch = [&](int32_t u, const Ids& e) {
            int32_t base, end;
            place(min(u, units - 1), base, end);
            seen = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int32_t key = base + h * 16 + col;
                const uint32_t id = e.low[h];
                const bool good = key < end && id >= 1 && id < a.pages && (a.table64 == 0 || e.high[h] == 0);
                const uint32_t inside = key - a.page.div(key) * a.page.divisor;
                const char* at = good ? a.keys + uint64_t{id} * a.page_stride + uint64_t{inside} * a.token_stride : nothing;
                const float* scale_at =
                    a.scales + (int64_t{id} * a.page.divisor + inside) * a.scale_step;
                scale[h] = *(good ? scale_at : reinterpret_cast<const float*>(nothing));
#pragma unroll
                for (int c = 0; c < kSteps; ++c) {
                    // Behind the key's last piece any other of its pieces: it meets codes of 0.
                    const int piece = (c * 4 + quad) * 16;
                    k[h][c] = *reinterpret_cast<const i32x4*>(at + (good && piece < a.dim ? piece : 0));
                }
                seen |= (static_cast<uint32_t>(__ballot(good)) & 0xffffu) << (16 * h);
            }
        };
        float best[kTiles];
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            best[m] = -INFINITY;
        }
        const auto leave = [&](int m, float score, int32_t block) {
            const float times = score > -INFINITY ? score * q_scale[m] : -INFINITY;
            if (pair_of[m] >= 0 && block < held) {
                atomicMax(&s_score[pair_of[m] * held + block], ordered(times));
            }
        };
        if (from < to) {
            Ids ids = ids_of(from);
            fetch(from, ids);
            ids = ids_of(from + 1);
#pragma unroll 1
            for (int32_t u = from; u < to; ++u) {
                const Ids later = ids_of(u + 2);
                int32_t base, end;
                place(u, base, end);
                const uint32_t now = seen;
                float key_scale[2][4];
                i32x4 s[kTiles][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        key_scale[h][j] = __shfl(scale[h], quad * 4 + j);
                    }
                }
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        s[m][h] = i32x4{0, 0, 0, 0};
#pragma unroll
                        for (int c = 0; c < kSteps; ++c) {
                            s[m][h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[h][c], q[m][c], s[m][h], 0, 0, 0);
                        }
                    }
                }
                fetch(u + 1, ids);
                ids = later;
                const bool ragged = now != 0xffffffffu || base + kUnit > first_seen;
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
                    float x[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            x[h][j] = static_cast<float>(s[m][h][j]) * key_scale[h][j];
                        }
                    }
                    if (ragged) {
                        const int32_t left = sight[m] - base;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int key = h * 16 + quad * 4 + j;
                                x[h][j] = ((now >> key) & 1) != 0 && key < left ? x[h][j] : -INFINITY;
                            }
                        }
                    }
                    if (a.sub_shift < 0) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                best[m] = fmaxf(best[m], x[h][j]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int32_t key = u * kUnit + h * 16 + quad * 4;      // from the segment's first
                            if (a.sub_shift == 0) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    leave(m, x[h][j], key + j);
                                }
                            } else if (a.sub_shift == 1) {
                                leave(m, fmaxf(x[h][0], x[h][1]), key >> 1);
                                leave(m, fmaxf(x[h][2], x[h][3]), (key >> 1) + 1);
                            } else {
                                leave(m, fmaxf(fmaxf(x[h][0], x[h][1]), fmaxf(x[h][2], x[h][3])), key >> a.sub_shift);
                            }
                        }
                    }
                }
                if (a.sub_shift < 0) {
                    const int32_t block = u / a.block_units;
                    if (u + 1 == to || (u + 1) / a.block_units != block) {
#pragma unroll
                        for (int m = 0; m < kTiles; ++m) {
                            const float most = over_quads_max(best[m]);
                            if (quad == 0) {
                                leave(m, most, block);
                            }
                            best[m] = -INFINITY;
                        }
                    }
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < pair_count * held; i += kThreads) {
            const int32_t pair = i / held, block = i - pair * held;
            a.scores[(int64_t{row.first} * a.groups + pair_begin + pair) * a.score_row + block_begin + block] = s_score[i];
        }
        __syncthreads();
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

    __device__ __forceinline__ uint32_t key(int32_t j) const {
        const uint32_t k = j < count ? scores[j] : 0u;
        return k != 0 && (j < forced_below || j >= forced_from) ? 0xffffffffu : k;
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
    return c;
}

// One wave a (token, group): block 64 r + lane in register r. The K-th largest key bit by bit, by counting the keys that
// are not below a bound; then the keys above it and the first of those equal to it, in order of their blocks.
template <int kRegs>
__global__ __launch_bounds__(kThreads) void pick_kernel(const PickArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t pair = int64_t{blockIdx.x} * kWaves + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    if (pair >= int64_t{a.at.tokens} * a.groups) {
        return;
    }
    const Candidates c = candidates_of(a, pair);
    uint32_t key[kRegs];
#pragma unroll
    for (int r = 0; r < kRegs; ++r) {
        key[r] = c.key(r * 64 + lane);
    }
    const auto not_below = [&](uint32_t bound) {
        int32_t n = 0;
#pragma unroll
        for (int r = 0; r < kRegs; ++r) {
            n += __popcll(__ballot(key[r] >= bound));
        }
        return n;
    };
    uint32_t bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t tried = bound | (1u << bit);
        const int32_t n = not_below(tried);
        if (n >= a.chosen) {
            bound = tried;
            if (n == a.chosen) {
                break;
            }
        }
    }
    int32_t equal = a.chosen - (bound == 0xffffffffu ? 0 : not_below(bound + 1));     // how many equal to the bound
    const int32_t token = a.group_div.div(static_cast<uint32_t>(pair)), group = static_cast<int32_t>(pair) - token * a.groups;
    int32_t* const out = a.blocks + token * a.b_token + group * a.b_group;
    int32_t at = 0;
#pragma unroll
    for (int r = 0; r < kRegs; ++r) {
        const uint64_t same = __ballot(bound != 0 && key[r] == bound);
        const uint64_t mine = uint64_t{1} << lane;
        const bool take = key[r] > bound || ((same & mine) != 0 && __popcll(same & (mine - 1)) < equal);
        const uint64_t taken = __ballot(take);
        if (take) {
            out[(at + __popcll(taken & (mine - 1))) * a.b_column] = r * 64 + lane;
        }
        at += __popcll(taken);
        equal -= min(equal, static_cast<int32_t>(__popcll(same)));
    }
    for (int32_t i = at + lane; i < a.chosen; i += 64) {
        out[i * a.b_column] = -1;
    }
}

constexpr int kManyThreads = 1024, kManyWaves = 16;

// The same by a workgroup, for any number of blocks: they are read again for every bit.
__global__ __launch_bounds__(kManyThreads) void pick_many_kernel(const PickArgs a) {
    __shared__ int32_t s_count[2][kManyWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t pair = blockIdx.x;
    const Candidates c = candidates_of(a, pair);
    int parity = 0;
    const auto total = [&](int32_t mine) {
        // mine: the wave's count, the same in all its lanes.
        s_count[parity][wave] = mine;
        __syncthreads();
        int32_t n = 0;
        for (int w = 0; w < kManyWaves; ++w) {
            n += s_count[parity][w];
        }
        parity ^= 1;
        return n;
    };
    const auto not_below = [&](uint32_t bound) {
        int32_t n = 0;
        for (int32_t j = tid; j - lane < c.count; j += kManyThreads) {
            n += __popcll(__ballot(c.key(j) >= bound));
        }
        return total(n);
    };
    uint32_t bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t tried = bound | (1u << bit);
        const int32_t n = not_below(tried);
        if (n >= a.chosen) {
            bound = tried;
            if (n == a.chosen) {
                break;
            }
        }
    }
    const int32_t equal = a.chosen - (bound == 0xffffffffu ? 0 : not_below(bound + 1));
    const int32_t token = a.group_div.div(static_cast<uint32_t>(pair)), group = static_cast<int32_t>(pair) - token * a.groups;
    int32_t* const out = a.blocks + token * a.b_token + group * a.b_group;
    int32_t at = 0, sames = 0;
    for (int32_t chunk = 0; chunk < c.count; chunk += kManyThreads) {
        const uint32_t key = c.key(chunk + tid);
        const uint64_t mine = uint64_t{1} << lane, below = mine - 1;
        const uint64_t same = __ballot(bound != 0 && key == bound), above = __ballot(key > bound);
        __syncthreads();
        s_count[0][wave] = __popcll(same);
        s_count[1][wave] = __popcll(above);
        __syncthreads();
        int32_t same_before = sames, above_before = 0, above_all = 0, same_all = 0;
        for (int w = 0; w < kManyWaves; ++w) {
            same_before += w < wave ? s_count[0][w] : 0;
            above_before += w < wave ? s_count[1][w] : 0;
            same_all += s_count[0][w], above_all += s_count[1][w];
        }
        const int32_t same_rank = same_before + __popcll(same & below);
        const int32_t taken_same = min(same_rank, equal) - min(sames, equal);
        const int32_t place = at + above_before + __popcll(above & below) + taken_same;
        if ((above & mine) != 0 || ((same & mine) != 0 && same_rank < equal)) {
            out[place * a.b_column] = chunk + tid;
        }
        at += above_all + min(sames + same_all, equal) - min(sames, equal);
        sames += same_all;
    }
    for (int32_t i = at + tid; i < a.chosen; i += kManyThreads) {
        out[i * a.b_column] = -1;
    }
}

// ---------------------------------------------------------------- host

constexpr int64_t kMostTokens = 1 << 23, kMostBatch = 1 << 20, kMostGroups = 1024, kMostShare = 128,
                  kMostPairs = 1 << 22;      // a workgroup each, of 1024 threads: fewer than 2^32 threads

struct Plan {
    int64_t score_row = 0;
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
        throw std::invalid_argument("more than 2^22 selections");
    }
    Plan p;
    p.score_row = std::max<int64_t>((columns * page_size + block_size - 1) / block_size, 1);
    p.bytes = (static_cast<uint64_t>(tokens * groups) * static_cast<uint64_t>(p.score_row) * 4 + 255) / 256 * 256;
    return p;
}

template <int kSteps>
void launch_scores(const ScoreArgs& a, int tiles16, uint32_t grid, uint32_t lds, hipStream_t stream) {
    switch (tiles16) {
        case 1: score_kernel<kSteps, 1><<<grid, kThreads, lds, stream>>>(a); break;
        case 2: score_kernel<kSteps, 2><<<grid, kThreads, lds, stream>>>(a); break;
        case 4: score_kernel<kSteps, 4><<<grid, kThreads, lds, stream>>>(a); break;
        default: score_kernel<kSteps, 8><<<grid, kThreads, lds, stream>>>(a); break;
    }
    check_hip(hipGetLastError(), "launch block scores");
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
    for (int d = 0; d < 3; ++d) {
        if (blocks.shape[d] > 1 && blocks.stride[d] == 0) {
            throw std::invalid_argument("blocks must not repeat its elements");
        }
    }
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
    if (workspace_bytes < plan.bytes) {
        throw std::invalid_argument("the selection needs " + std::to_string(plan.bytes) + " workspace bytes, got " +
                                    std::to_string(workspace_bytes));
    }
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0) {
        throw std::invalid_argument("the workspace must be a 256-byte aligned device buffer");
    }
    if (tokens == 0) {
        return 0;
    }
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
    a.block_units = static_cast<int32_t>((s.block_size + kUnit - 1) / kUnit);
    a.sub_shift = -1;
    for (int shift = 0; shift < 5; ++shift) {
        if (s.block_size == 1 << shift) {
            a.sub_shift = shift;
        }
    }
    a.scores = static_cast<uint32_t*>(workspace);
    a.score_row = plan.score_row;
    const int64_t most_rows = std::min(s.max_query, tokens) * heads;
    int tiles16 = most_rows <= 16 ? 1 : (most_rows <= 32 ? 2 : (most_rows <= 64 ? 4 : 8));
    while (16 * tiles16 < a.share) {
        tiles16 *= 2;
    }
    a.pairs = 16 * tiles16 / a.share;
    a.row_tiles = (a.groups + a.pairs - 1) / a.pairs;
    a.tiles = static_cast<int32_t>(s.query_starts != nullptr ? tokens * groups / a.pairs + a.at.batch
                                                             : tokens * a.row_tiles);
    // Segments of at least 256 tokens, longer where the context makes more than 2048 workgroups, and as many blocks as
    // there is room for keys.
    const int64_t capacity = std::max<int64_t>(a.at.own_most, 1);
    int64_t wanted = std::min<int64_t>(std::max<int64_t>(a.tiles * capacity / 2048, 256), 4096);
    wanted = (wanted + kUnit - 1) / kUnit * kUnit;
    int64_t segment_blocks = std::max<int64_t>(wanted / s.block_size, 1);
    segment_blocks = std::min<int64_t>(segment_blocks, kSegmentKeys / a.pairs);
    if (a.sub_shift >= 0) {
        segment_blocks = std::max<int64_t>(segment_blocks >> (5 - a.sub_shift), 1) << (5 - a.sub_shift);
    }
    a.segment_blocks = static_cast<int32_t>(segment_blocks);
    int64_t segments = std::min<int64_t>((plan.score_row + segment_blocks - 1) / segment_blocks,
                                         std::max<int64_t>(65536 / a.tiles, 1));
    if (segments > 8) {
        segments = (segments + 7) / 8 * 8;
    }
    a.segments = static_cast<int32_t>(segments);
    const uint32_t lds = static_cast<uint32_t>(a.pairs * segment_blocks * 4);
    const auto on = static_cast<hipStream_t>(stream);
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
    const uint32_t pairs = static_cast<uint32_t>(tokens * groups), grid = (pairs + kWaves - 1) / kWaves;
    if (plan.score_row <= 64) {
        pick_kernel<1><<<grid, kThreads, 0, on>>>(k);
    } else if (plan.score_row <= 256) {
        pick_kernel<4><<<grid, kThreads, 0, on>>>(k);
    } else if (plan.score_row <= 1024) {
        pick_kernel<16><<<grid, kThreads, 0, on>>>(k);
    } else {
        pick_many_kernel<<<pairs, kManyThreads, 0, on>>>(k);
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
