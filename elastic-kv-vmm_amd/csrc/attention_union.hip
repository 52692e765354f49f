// Attention of prompts' query tokens to the blocks that each lists: neighbouring tokens list mostly the same blocks, so a
// workgroup takes 64 query rows (tokens x query heads of a KV head) and goes once through all blocks that any of its tokens
// lists (gfx950).
//
// First it makes that list: a word of 64 bits for each block of the context in LDS, bit t for the tile's t-th token, and
// then the blocks whose word is not 0, in order, with their words. (A block that a token lists again goes into another
// round, and is in the list again: it counts twice.) Then it works as the kernel for many rows does: 32 keys down and 32
// rows across in 32x32x16 products, running largest score and sum, K and V of the next tile of 64 keys going into the other
// of two LDS buffers. Of a tile's 64 keys two waves take the first half for their 32 rows each, two the second, and the
// halves' sums are joined at the end. A row whose token does not list a block, or is not past all of its tokens, has those
// scores cut.
//
// What bounds it: each workgroup's chain of tiles, barrier, LDS, products and softmax one after the other with two waves
// on a SIMD. Four pieces of up to 512 tokens of 16 heads on 2 KV heads of 128, 16 blocks of 128 a list, take 91 us, token
// by token 432: 432 workgroups of 18 blocks together on average, the longest of 23, so that some compute units have two
// and some one: they have work 69 % of the time, the matrix pipes 13 and vector instructions 31 % of the cycles. 0.57 GB
// come from L2, nine tenths of them hits. Tried: 48 of the 290 vector instructions of a tile less, no change; 128 rows a
// workgroup, 102 us.
//
// The weights are rounded once to the inputs' type, as there.
#include "ekv_attention_wide.h"

namespace ekv {
namespace {

using wide::kTile;
using wide::over_halves_max;
using wide::over_halves_sum;
using wide::Tile;

constexpr int kThreads = 256, kWaves = 4, kRows = 64;

template <typename T, int kDim>
__global__ __launch_bounds__(kThreads, kDim <= 128 ? 2 : 1) void union_kernel(const Launch) {
    constexpr int kSteps = kDim / 16;              // matrix steps of the first product
    constexpr int kCols = kDim / 32;               // 32-column pieces of the output
    constexpr int kBytes = Tile<kDim>::kBytes;
    constexpr int kRowThreads = kBytes / 16;       // threads that load a key's row
    constexpr int kKeysAtOnce = kThreads / kRowThreads;
    constexpr int kLoads = kTile / kKeysAtOnce;
    static_assert(kUnionBlocks * 8 <= wide::lds_bytes<kDim>(), "the words of all blocks fit where the keys will be");
    __shared__ __align__(16) char s_data[wide::lds_bytes<kDim>()];
    __shared__ uint64_t s_mask[kUnionEntries];     // the tokens that list it
    __shared__ uint32_t s_block[kUnionEntries];
    __shared__ uint32_t s_cells[kWaves];
    __shared__ uint32_t s_spoiled[2];              // number + 1 of the last tile in each buffer whose V is not all finite
    __shared__ float s_top[kRows], s_sum[kRows];
    const char* const zeros = reinterpret_cast<const char*>(zero_row);
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row_half = wave & 1, key_half = wave >> 1;

    {
        // Tokens of no batch row are in front of the others and behind.
        const AttentionArgs& a = fresh().a;
        const int32_t front = a.batch > 0 ? first_token(a, 0) : 0, behind = a.batch > 0 ? first_token(a, a.batch) : 0;
        const int32_t gap = front + a.tokens - behind, pieces = a.dim >> 3;
        for (int32_t i = blockIdx.x; i < gap; i += gridDim.x) {
            const int32_t token = i < front ? i : behind + i - front;
            for (int32_t unit = tid; unit < a.heads * pieces; unit += kThreads) {
                const int32_t head = unit / pieces, piece = unit - head * pieces;
                *reinterpret_cast<words4*>(a.out + token * a.o_token + head * a.o_head + piece * 16) = words4{0, 0, 0, 0};
                if (piece == 0 && a.lse != nullptr) {
                    a.lse[token * a.l_token + head * a.l_head] = -INFINITY;
                }
            }
        }
    }

    // The tile: KV head, batch row, query rows row_begin .. of it.
    int32_t head, first, rows, row_begin, position, seen_most, request;
    {
        const Launch& l = fresh();
        const AttentionArgs& a = l.a;
        // Tiles of a head lie side by side: their blocks meet behind one L2.
        const int32_t item = on_die(blockIdx.x, gridDim.x);
        head = uniform(item / l.lists.tiles);
        const int32_t tile = item - head * l.lists.tiles;
        // Batch row b has tiles from starts[b] * share / 64 + b on.
        const auto begin = [&](int32_t b) {
            return static_cast<int32_t>(static_cast<int64_t>(first_token(a, b)) * a.share / kRows) + b;
        };
        int32_t low = 0, high = a.batch;
        while (high - low > 1) {
            const int32_t mid = (low + high) >> 1;
            const bool here = begin(mid) <= tile;
            low = here ? mid : low;
            high = here ? high : mid;
        }
        if (a.batch == 0) {
            return;
        }
        const int32_t part = tile - begin(low);
        first = first_token(a, low);
        const int32_t count = max(first_token(a, low + 1) - first, 0);
        rows = count * a.share, row_begin = part * kRows;
        if (part < 0 || row_begin >= rows) {
            return;
        }
        const int64_t length = a.lengths.fetch(low), given = a.rows.data != nullptr ? a.rows.fetch(low) : low;
        const bool good = given >= 0 && given < a.requests;
        request = uniform(good ? static_cast<int32_t>(given) : 0);
        seen_most = uniform(good ? clamped(length, 0, a.block_most) : 0);
        position = uniform(clamped(length, -1, 0x7ffffffe) - count);
        first = uniform(first), rows = uniform(rows), row_begin = uniform(row_begin);
    }
    // Tokens that the batch row's i-th query token sees.
    const auto seen_by_token = [&](int32_t i) { return min(max(position + i + 1, 0), seen_most); };
    const FastDiv share_div = fresh().a.share_div, block = fresh().lists.block;
    const int32_t token_begin = share_div.div(row_begin);
    const int32_t tokens = static_cast<int32_t>(share_div.div(min(row_begin + kRows, rows) - 1)) - token_begin + 1;
    const int32_t last_seen = seen_by_token(token_begin + tokens - 1);
    const int32_t blocks = last_seen > 0 ? block.div(last_seen - 1) + 1 : 0;

    // The blocks that some token lists.
    int32_t entries = 0;
    {
        const BlockLists& lists = fresh().lists;
        uint64_t* const words = reinterpret_cast<uint64_t*>(s_data);
        int32_t id[kUnionEntries / kThreads], by[kUnionEntries / kThreads];
#pragma unroll
        for (int k = 0; k < kUnionEntries / kThreads; ++k) {
            const int32_t i = tid + k * kThreads;
            id[k] = -1;
            by[k] = i / lists.width;
            if (i < tokens * lists.width) {
                const char* at = lists.lists + (first + token_begin + by[k]) * lists.token +
                                 static_cast<int64_t>(lists.heads.div(head)) * lists.group +
                                 static_cast<uint64_t>(i - by[k] * lists.width) * lists.column;
                const uint32_t low = load_global<uint32_t>(at), high = load_global<uint32_t>(at + lists.wide);
                const int32_t seen = seen_by_token(token_begin + by[k]);
                const uint32_t there = seen > 0 ? block.div(seen - 1) + 1 : 0;
                id[k] = low < there && (lists.wide == 0 || high == 0) ? static_cast<int32_t>(low) : -1;
            }
        }
        if (tid < 2) {
            s_spoiled[tid] = 0;
        }
        bool again;
        do {
            for (int32_t i = tid; i < blocks; i += kThreads) {
                words[i] = 0;
            }
            __syncthreads();
            again = false;
#pragma unroll
            for (int k = 0; k < kUnionEntries / kThreads; ++k) {
                if (id[k] >= 0) {
                    const unsigned long long bit = 1ull << by[k];
                    const unsigned long long old = atomicOr(reinterpret_cast<unsigned long long*>(words + id[k]), bit);
                    again |= (old & bit) != 0;
                    id[k] = (old & bit) != 0 ? id[k] : -1;
                }
            }
            __syncthreads();
            for (int32_t i = 0; i < blocks; i += kThreads) {
                const uint64_t word = i + tid < blocks ? words[i + tid] : 0;
                const uint64_t taken = __ballot(word != 0);
                if (lane == 0) {
                    s_cells[wave] = __popcll(taken);
                }
                __syncthreads();
                int32_t at = entries;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const int32_t n = __builtin_amdgcn_readfirstlane(static_cast<int>(s_cells[w]));
                    at += w < wave ? n : 0;
                    entries += n;
                }
                at += __popcll(taken & ((uint64_t{1} << lane) - 1));
                if (word != 0 && at < kUnionEntries) {
                    s_block[at] = i + tid, s_mask[at] = word;
                }
                __syncthreads();
            }
        } while (__syncthreads_or(again));
        entries = uniform(min(entries, kUnionEntries));
    }

    const AttentionArgs& a = fresh().a;
    const int pieces = a.dim >> 3;
    const float scale = a.scale, slack = kSlack / fmaxf(a.scale, 1e-30f);
    const int32_t row = row_begin + row_half * 32 + col;           // the lane's query row
    const bool live = row < rows;
    const int32_t token = share_div.div(row), in_share = row - token * a.share;
    const int32_t place = live ? token - token_begin : 0;          // its bit
    const int32_t my_seen = live ? seen_by_token(token) : 0x7fffffff;
    words4 q[kSteps];
    {
        const char* at = a.query + (first + token) * a.q_token + (head * a.share + in_share) * a.q_head;
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            const int piece = c * 2 + half;
            q[c] = load_global<words4>(live && piece < pieces ? at + piece * 16 : zeros);
            q[c] ^= a.flip;
        }
    }
    f32x16 o[kCols];
    float top = -INFINITY, sum = 0;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            o[c][i] = 0;
        }
    }

    // Runs of 32 keys: `runs_of` to a block, whose last may be part-filled; two to a tile.
    const FastDiv runs_of = fresh().lists.runs_of;
    const int32_t runs = entries * static_cast<int32_t>(runs_of.divisor), tiles = (runs + 1) >> 1;
    if (tiles > 0) {
        const Cache cache = a.cache;
        const char* const table = a.tables + request * a.table_row;
        const uint32_t step = a.table_col, wide64 = a.table64 != 0 ? 4 : 0;
        const int load_key = tid / kRowThreads, load_piece = tid % kRowThreads;
        const int write_at = Tile<kDim>::place(load_key, load_piece);
        const int read_k = Tile<kDim>::place(col, half);
        const int v_key = half * 4 + ((lane & 15) >> 2), v_piece = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
        const int read_v = Tile<kDim>::kSize + Tile<kDim>::place(v_key, v_piece) + (lane & 1) * 8;
        const int read_v8 = Tile<kDim>::kSize + Tile<kDim>::place(v_key + 8, v_piece) + (lane & 1) * 8;
        const int half_at = key_half * 32 * kBytes;                // of a tile, the wave's keys
        const char* const k_head = cache.k + static_cast<uint64_t>(cache.head_stride) * head +
                                   (load_piece < pieces ? load_piece : 0) * 16;

        // Page id of a tile's key `lane`, and its place in the page (~0: nobody sees it).
        struct Ids {
            uint32_t low, high, inside;
        };
        const auto ids_of = [&](int32_t tile) {
            const int32_t run = 2 * tile + half;
            const bool there = run < runs;
            const int32_t entry = there ? static_cast<int32_t>(runs_of.div(run)) : 0;
            const int32_t in_block = (run - entry * static_cast<int32_t>(runs_of.divisor)) * 32 + col;
            const int32_t key = static_cast<int32_t>(s_block[entry] * block.divisor) + in_block;
            const bool good = there && in_block < static_cast<int32_t>(block.divisor) && key < last_seen;
            const uint32_t page = cache.page.div(key);
            const char* at = good ? table + static_cast<uint64_t>(page) * step : zeros;
            return Ids{load_global<uint32_t>(at), load_global<uint32_t>(at + wide64),
                       good ? key - page * cache.page.divisor : ~0u};
        };
        uint32_t offset_low = 0, offset_high = 0;                  // of key `lane` of the tile to be loaded
        const auto look = [&](const Ids& ids) {
            const bool good = ids.inside != ~0u && ids.low >= cache.zero_below && ids.low < cache.pages &&
                              (wide64 == 0 || ids.high == 0);
            const uint64_t offset = static_cast<uint64_t>(ids.low) * cache.page_stride +
                                    static_cast<uint64_t>(ids.inside) * cache.token_stride;
            offset_low = good ? static_cast<uint32_t>(offset) : ~0u;
            offset_high = good ? static_cast<uint32_t>(offset >> 32) : ~0u;
            return __ballot(good);
        };
        words4 k[kLoads], v[kLoads];                               // a tile's rows on their way to LDS
        const auto load = [&] {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t low = __shfl(offset_low, i * kKeysAtOnce + load_key);
                const uint32_t high = __shfl(offset_high, i * kKeysAtOnce + load_key);
                const char* at = k_head + (static_cast<uint64_t>(high) << 32 | low);
                const char* v_at = at + cache.kv_stride;
                k[i] = load_global<words4>(high != ~0u ? at : zeros);
                v[i] = load_global<words4>(high != ~0u ? v_at : zeros);
            }
        };
        const auto store = [&](int buffer, int32_t tile) {
            typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
            u16x2 most = {0, 0};
            const int at = hidden(write_at);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                char* const to = s_data + buffer + i * kKeysAtOnce * kBytes + (at ^ ((i * kKeysAtOnce & 8) << 2));
                // K past the head size meets zeros of q and must not be an infinity; V's columns are not stored.
                *reinterpret_cast<words4*>(to) = load_piece < pieces ? k[i] : words4{0, 0, 0, 0};
                *reinterpret_cast<words4*>(to + Tile<kDim>::kSize) = v[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, v[i][e] & 0x7fff7fffu));
                }
            }
            constexpr uint16_t kExponent = static_cast<uint16_t>(T::kExponent);
            if (__ballot(most[0] >= kExponent || most[1] >= kExponent) != 0) {
                s_spoiled[tile & 1] = tile + 1;
            }
        };
        // Of the wave's 32 keys of a tile: which there are, and how many of them the lane's row sees.
        uint32_t bits = 0;
        int32_t left = 0;
        const auto sight = [&](int32_t tile, uint64_t now) {
            const int32_t run = 2 * tile + key_half;
            const int32_t entry = run < runs ? static_cast<int32_t>(runs_of.div(run)) : 0;
            const int32_t base = static_cast<int32_t>(s_block[entry] * block.divisor) +
                                 (run - entry * static_cast<int32_t>(runs_of.divisor)) * 32;
            const bool listed = !live || ((s_mask[entry] >> place) & 1) != 0;
            left = listed ? min(max(my_seen - base, 0), 32) : 0;
            bits = static_cast<uint32_t>(now >> (32 * key_half));
            return __ballot(left < 32) == 0 && bits == 0xffffffffu;
        };
        const auto cut_scores = [&](f32x16& s) {
            rarely();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = half * 4 + (i & 3) + 8 * (i >> 2);
                s[i] = ((bits >> key) & 1) != 0 && key < left ? s[i] : -INFINITY;
            }
        };
        const auto largest = [&](const f32x16& s) {
            float most = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) {
                most = fmaxf(most, s[i]);
            }
            return over_halves_max(most);
        };
        // The reference score follows the largest only when that has passed it by 2^kSlack: until then the weights are
        // larger than 1, which their type holds, and nothing has to be scaled again.
        const auto follow = [&](float most) {
            if (__ballot(most > top + slack) != 0) {
                const float to_top = fmaxf(top, most);
                const float keep = to_top == top ? 1.0f : __builtin_amdgcn_exp2f((top - to_top) * scale);
                sum *= keep;
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    o[c] *= keep;
                }
                top = to_top;
            }
        };
        // The rows of a tile leave their registers for LDS while the tile before it is worked on, the next one's are then
        // on their way, and the page ids of the one after that. One barrier a tile; products and softmax of a wave stand
        // beside those of the other workgroup on the compute unit.
        uint64_t now, next;
        Ids ids;
        {
            const Ids first_ids = ids_of(0), second_ids = ids_of(1);
            ids = ids_of(2);
            now = look(first_ids);
            load();
            store(0, 0);
            next = look(second_ids);
            load();
        }
        int buffer = 0;
#pragma unroll 1
        for (int32_t tile = 0; tile < tiles; ++tile, buffer ^= 2 * Tile<kDim>::kSize) {
            lds_barrier();      // this buffer holds the tile, and nobody reads the other one any more
            const char* const here = s_data + buffer;
            // Hidden, or what follows from them would be computed once and spilled.
            const int at_k = hidden(read_k), at_v = hidden(read_v), at_v8 = hidden(read_v8);
            store(buffer ^ (2 * Tile<kDim>::kSize), tile + 1);
            const bool whole = sight(tile, now);
            now = next;
            {
                const Ids later = ids_of(tile + 3);      // before the rows: a wait for them would be for the rows as well
                next = look(ids);
                load();
                ids = later;
            }
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = 0;
            }
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                s = T::mfma32(*reinterpret_cast<const words4*>(here + (at_k ^ (c << 5)) + half_at), q[c], s);
            }
            if (!whole) {
                cut_scores(s);
            }
            follow(largest(s));
            if (s_spoiled[tile & 1] == static_cast<uint32_t>(tile + 1)) {
                // A key that only some rows see has weight 0 for the others, and 0 * infinity is not 0: the infinities
                // and NaN are added to the rows that see them (a weight is positive), then cleared.
                rarely();
                const int my_half = hidden(half);
#pragma unroll 1
                for (int key = 0; key < 32; ++key) {
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const words2 x = *reinterpret_cast<const words2*>(
                                here + half_at + Tile<kDim>::kSize + Tile<kDim>::place(key, c * 4 + (i >> 2)) + my_half * 8);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                o[c][i + e] += key < left ? T::unbounded(x[e >> 1] >> (16 * (e & 1))) : 0.0f;
                            }
                        }
                    }
                }
                lds_barrier();
#pragma unroll 1
                for (int at = hidden(tid) * 16; at < Tile<kDim>::kSize; at += kThreads * 16) {
                    words4* const to = reinterpret_cast<words4*>(s_data + buffer + Tile<kDim>::kSize + at);
                    words4 x = *to;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = bounded<T>(x[e]);
                    }
                    *to = x;
                }
                lds_barrier();
            }
            const float shift = (top == -INFINITY ? 0.0f : top * scale) - T::kShift;
            words4 weights[2];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float x = __builtin_amdgcn_exp2f(s[i] * scale - shift);
                const float y = __builtin_amdgcn_exp2f(s[i + 1] * scale - shift);
                sum += x;
                sum += y;
                weights[i >> 3][(i & 7) >> 1] = T::pack(x, y);
            }
#pragma unroll
            for (int j = 0; j < 2 * kCols; ++j) {     // 16 keys, 32 columns
                const int at = half_at + j / kCols * 16 * kBytes;
                const words2 low = read_transposed(here + (at_v ^ (j % kCols << 6)) + at);
                const words2 high = read_transposed(here + (at_v8 ^ (j % kCols << 6)) + at);
                o[j % kCols] = T::mfma32(words4{low[0], low[1], high[0], high[1]}, weights[j / kCols], o[j % kCols]);
            }
        }
    }

    // The two halves of the keys, joined.
    sum = over_halves_sum(sum);
    top = top == -INFINITY ? top : top * scale;
    f32x4* const joined = reinterpret_cast<f32x4*>(s_data) + row_half * (kCols * 4 * 64);
    __syncthreads();
    if (key_half == 1) {
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                joined[(c * 4 + (i >> 2)) * 64 + lane] = f32x4{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]};
            }
        }
        if (half == 0) {
            s_top[row_half * 32 + col] = top, s_sum[row_half * 32 + col] = sum;
        }
    }
    __syncthreads();
    if (key_half == 0 && live) {
        const AttentionArgs& z = fresh().a;
        const float other_top = s_top[row_half * 32 + col], all = fmaxf(top, other_top);
        const float safe = all == -INFINITY ? 0.0f : all;
        const float mine = __builtin_amdgcn_exp2f(top - safe), theirs = __builtin_amdgcn_exp2f(other_top - safe);
        const float total = sum * mine + s_sum[row_half * 32 + col] * theirs;
        const float inverse = total == 0 ? 0.0f : 1.0f / total;
        char* const to = z.out + (first + token) * z.o_token + (head * z.share + in_share) * z.o_head;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int element = c * 32 + half * 4 + 2 * i;
                const f32x4 y = joined[(c * 4 + (i >> 2)) * 64 + lane];
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = (o[c][i + e] * mine + y[e] * theirs) * inverse;
                }
                if (element < z.dim) {
                    *reinterpret_cast<words2*>(to + element * 2) = words2{T::pack(x[0], x[1]), T::pack(x[2], x[3])};
                }
            }
        }
        if (half == 0 && z.lse != nullptr) {
            z.lse[(first + token) * z.l_token + (head * z.share + in_share) * z.l_head] =
                total == 0 ? -INFINITY : (all - T::kShift + log2f(total)) * kLn2;
        }
    }
}

template <typename T>
void launch_type(const Launch& l, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(l.lists.tiles) * l.a.kv_heads);
    switch (l.p[0].dim_pad) {
        case 64: union_kernel<T, 64><<<grid, kThreads, 0, stream>>>(l); break;
        case 96: union_kernel<T, 96><<<grid, kThreads, 0, stream>>>(l); break;
        case 128: union_kernel<T, 128><<<grid, kThreads, 0, stream>>>(l); break;
        default: union_kernel<T, 256><<<grid, kThreads, 0, stream>>>(l); break;
    }
    check_hip(hipGetLastError(), "launch block attention");
}

}  // namespace

void launch_union(const Launch& l, int32_t dtype, void* stream) {
    if (dtype == EKV_BFLOAT16) {
        launch_type<Bf16>(l, static_cast<hipStream_t>(stream));
    } else {
        launch_type<F16>(l, static_cast<hipStream_t>(stream));
    }
}

}  // namespace ekv
