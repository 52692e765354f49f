// Attention of many query rows to the same keys: a large batch against its shared prefix, prompt pieces against prefix
// and own tokens (gfx950).
//
// Mathematics, per wave of 32 query rows and 32 keys: S^T = K Q^T by 32x32x16 matrix instructions (keys down, rows
// across: a lane holds 16 scores of one row, its other half-wave the other 16), running largest score and sum per row,
// P^T = exp(S^T - m) rounded once to 16 bits, O^T += V^T P^T. As in the kernel for few rows, P stays in the registers
// that the first product left it in, and the transposed LDS read gives V^T in the same order of keys.
//
// What bounds it: the matrix pipes, the softmax beside them and the LDS that feeds them. A workgroup's waves share each
// tile of 64 keys: K and V of the next tile go from registers into the other of two LDS buffers, and the one after's
// rows are loaded, while a tile is worked on; one barrier a half tile. At a head size of 128 a half tile is 16 KB of LDS
// reads, 16 matrix instructions (512 cycles) and about as many cycles of vector instructions a wave, dealt in turn.
//
// The weights are rounded once to the inputs' type, as there.
//
// Measured: prompts of 0.96 TFLOP, head size 128, bfloat16, 256 rows a workgroup: 1.06 ms, 0.91 PFLOP/s (a library
// product of 16384^3 reaches 1.33); the matrix pipes are busy 47 % of the cycles at the 1.8 GHz that the card holds
// under this load, LDS 31 %, with no bank conflicts. Staged between the tiles instead of beside the products it took
// 1.13 ms. 128 rows a workgroup read the keys twice as often: two workgroups of four waves a compute unit, which
// smaller batches fill better.
#pragma once

#include "ekv_attention.h"
#include "ekv_mfma.h"

namespace ekv {
namespace wide {

constexpr int kTile = 64;   // keys of a tile

template <int kDim>
struct Tile {
    static constexpr int kBytes = kDim <= 64 ? 128 : (kDim <= 128 ? 256 : 512);   // of a row in LDS
    static constexpr int kPieces = kDim / 8;
    static constexpr int kSize = kTile * kBytes;
    // The 16-byte pieces of a row are permuted by exclusive or so that 16 lanes with 16 keys and one piece (K) and the
    // four rows of 64 bytes that a transposed read takes at a time (V) each meet every bank once.
    // The permutation depends on key % 16 alone, so other keys and pieces are offsets and exclusive ors of one address.
    static __device__ __forceinline__ int place(int key, int piece) {
        const int swap = kBytes == 128 ? (((key >> 1) & 1) << 2) | ((key >> 2) & 3) : ((key & 3) << 2) | ((key >> 2) & 3);
        return key * kBytes + ((piece ^ swap) << 4);
    }
};

__device__ __forceinline__ float over_halves_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ float over_halves_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

template <int kDim>
constexpr int lds_bytes() {
    return 4 * Tile<kDim>::kSize;      // two buffers of K and V
}

// Workgroup w's part of phase `which` of the launch. s_data: lds_bytes() of LDS.
template <typename T, int kDim, int kWaves, int kChunk>
__device__ __forceinline__ void run(int which, uint32_t w, uint32_t workgroups, bool read, uint32_t total,
                                    char* s_data, LineCells<kWaves, kChunk>& cells) {
    constexpr int kSteps = kDim / 16;              // matrix steps of the first product
    constexpr int kCols = kDim / 32;               // 32-column pieces of the output
    constexpr int kRowThreads = Tile<kDim>::kBytes / 16;               // threads that load a key's row
    constexpr int kKeysAtOnce = kWaves * 64 / kRowThreads;
    constexpr int kLoads = kTile / kKeysAtOnce;    // 16-byte pieces of K, and of V, that a thread loads a tile
    static_assert(kLoads >= 1, "a tile has at least one piece for every thread");
    static_assert(kKeysAtOnce % 8 == 0, "8 keys on, a row's permutation differs by 2");
    constexpr int kBytes = Tile<kDim>::kBytes;
    const char* const zeros = reinterpret_cast<const char*>(zero_row);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));

    for_segments(which, w, workgroups, read, total, cells, [&](const Segment& g) {
        const int tid = hidden(threadIdx.x), lane = tid & 63, col = lane & 31, half = lane >> 5;
        const int load_key = tid / kRowThreads, load_piece = tid % kRowThreads;
        const int write_at = Tile<kDim>::place(load_key, load_piece);
        // K of key col, piece half; V^T of 16 keys and 32 columns: lane (half, 16-column piece, i) names row 4 half + i / 4
        // (and + 8), the (i % 4)-th 8 bytes of its 32.
        const int read_k = Tile<kDim>::place(col, half);
        const int v_key = half * 4 + ((lane & 15) >> 2), v_piece = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
        const int read_v = Tile<kDim>::kSize + Tile<kDim>::place(v_key, v_piece) + (lane & 1) * 8;
        const int read_v8 = Tile<kDim>::kSize + Tile<kDim>::place(v_key + 8, v_piece) + (lane & 1) * 8;
        const AttentionArgs& a = fresh().a;
        const int pieces = a.dim >> 3;
        const float slack = kSlack / fmaxf(a.scale, 1e-30f);     // in raw scores
        const int32_t row = g.row_begin + wave * 32 + col;     // the lane's query row
        const int32_t token = a.share_div.div(row), head = (g.head - token) * a.share + row;
        words4 q[kSteps];
        {
            const char* at = a.query + (g.q.first + token) * a.q_token + head * a.q_head;
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                const int piece = c * 2 + half;
                q[c] = load_global<words4>(row < g.rows && piece < pieces ? at + piece * 16 : zeros);
                q[c] ^= a.flip;
            }
        }
        const int32_t visible = seen_by(g.q, token);
        const int32_t first_visible = seen_by(g.q, a.share_div.div(g.row_begin));
        const int32_t last_row = min(g.row_begin + 32 * kWaves, g.rows) - 1;
        const int32_t last_visible = seen_by(g.q, a.share_div.div(last_row));

        f32x16 o[kCols];
        float top = -INFINITY, sum = 0;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                o[c][i] = 0;
            }
        }

        const int32_t unit_shift = fresh().p[which].unit_shift;
        const int32_t prefix_end = (g.q.prefix + (1 << unit_shift) - 1) >> unit_shift;
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
            const bool own = side == 1;
            const int32_t from = own ? max(g.begin - prefix_end, 0) : g.begin;
            const int32_t to = own ? g.end - prefix_end : min(g.end, prefix_end);
            if (to <= from) {
                continue;
            }
            const char* const table =
                own ? a.tables + g.q.request * a.table_row : a.prefix_tables + g.q.group * a.prefix_row;
            const uint32_t step = own ? a.table_col : a.prefix_col;
            const uint32_t wide = (own ? a.table64 : a.prefix64) != 0 ? 4 : 0;
            // Keys past the last that any row sees are nobody's.
            const int32_t keys = min(own ? last_visible : g.q.prefix, to << unit_shift);
            const char* const k_head = a.cache.k + static_cast<uint64_t>(a.cache.head_stride) * g.head +
                                       (load_piece < pieces ? load_piece : 0) * 16;

            const Cache cache = a.cache;

            // Page id of key base + lane, as words (an int64 id whose high word is not zero names no page): every wave
            // holds all of a tile's, and looks at them one tile later.
            struct Ids {
                uint32_t low, high;
            };
            const auto ids_of = [&](int32_t base) {
                const int32_t key = base + lane;
                const char* at = table + static_cast<uint64_t>(cache.page.div(key)) * step;
                at = key < keys ? at : zeros;
                return Ids{load_global<uint32_t>(at), load_global<uint32_t>(at + wide)};
            };
            words4 k[kLoads], v[kLoads];
            // A tile's rows in three parts: whose keys are seen, then piece i of its loads, then piece i of its stores.
            uint32_t mine = 0;
            const auto look = [&](int32_t base, const Ids& ids) {
                const bool good = base + lane < keys && ids.low >= cache.zero_below && ids.low < cache.pages &&
                                  (wide == 0 || ids.high == 0);
                mine = good ? ids.low : 0xffffffffu;
                return __ballot(good);
            };
            const auto load = [&](int32_t base, int i) {
                const int32_t inside_tile = i * kKeysAtOnce + load_key;
                const uint32_t id = __shfl(mine, inside_tile);
                const int32_t key = base + inside_tile;
                const uint32_t inside = key - cache.page.div(key) * cache.page.divisor;
                const char* at = k_head + static_cast<uint64_t>(id) * cache.page_stride +
                                 static_cast<uint64_t>(inside) * cache.token_stride;
                const char* v_at = at + cache.kv_stride;
                at = id != 0xffffffffu ? at : zeros;
                v_at = id != 0xffffffffu ? v_at : zeros;
                k[i] = load_global<words4>(at);
                v[i] = load_global<words4>(v_at);
            };
            const auto store = [&](int buffer, int i) {
                char* const to = s_data + buffer + i * kKeysAtOnce * kBytes + (write_at ^ ((i * kKeysAtOnce & 8) << 2));
                // K past the head size meets zeros of q and must not be an infinity; V's columns are not stored.
                const words4 kept = load_piece < pieces ? k[i] : words4{0, 0, 0, 0};
                *reinterpret_cast<words4*>(to) = kept;
                *reinterpret_cast<words4*>(to + Tile<kDim>::kSize) = v[i];
            };
            const auto load_all = [&](int32_t base) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    load(base, i);
                }
            };
            const auto store_all = [&](int buffer) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    store(buffer, i);
                }
            };
            const auto any_not_finite = [&](const char* tile, int first) {
                bool found = false;
#pragma unroll 1
                for (int at = first * 16; at < Tile<kDim>::kSize; at += 64 * 16) {
                    const words4 x = *reinterpret_cast<const words4*>(tile + Tile<kDim>::kSize + at);
                    found |= not_finite<T>(x[0]) || not_finite<T>(x[1]) || not_finite<T>(x[2]) || not_finite<T>(x[3]);
                }
                return __ballot(found) != 0;
            };

            // Scores of 32 keys of the tile at `tile`: its first or second half.
            const auto scores = [&](const char* tile, int b) {
                f32x16 s;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = 0;
                }
#pragma unroll
                for (int c = 0; c < kSteps; ++c) {
                    const words4 x = *reinterpret_cast<const words4*>(tile + (read_k ^ (c << 5)) + b * 32 * kBytes);
                    s = T::mfma32(x, q[c], s);
                }
                return s;
            };
            // Scores of the keys that a row does not see become -infinity; `left` keys of the 32 are before its end.
            const auto cut_scores = [&](f32x16& s, uint32_t bits, int32_t left) {
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
                    const float keep = to_top == top ? 1.0f : __builtin_amdgcn_exp2f((top - to_top) * a.scale);
                    sum *= keep;
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        o[c] *= keep;
                    }
                    top = to_top;
                }
            };
            // One step: the weights of s (32 keys, half b of `tile`) and their values, while the next step's scores, of
            // half `next_b` of `next_tile`, are multiplied: s becomes them. The matrix and the vector instructions are
            // dealt in turn, so that a wave's softmax runs beside its own products.
            const auto step_on = [&](f32x16& s, const char* tile, int b, const char* next_tile, int next_b, bool whole,
                                     uint32_t bits, int32_t left, auto&& beside) {
                const float shift = (top == -INFINITY ? 0.0f : top * a.scale) - T::kShift;
                f32x16 n;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    n[i] = 0;
                }
                const auto key_piece = [&](int c) {
                    return *reinterpret_cast<const words4*>(next_tile + (read_k ^ (c << 5)) + next_b * 32 * kBytes);
                };
                const auto column = [&](int j) {          // of 16-key group j / kCols, columns j % kCols
                    const int at = (b * 2 + j / kCols) * 16 * kBytes;
                    const words2 low = read_transposed(tile + (read_v ^ (j % kCols << 6)) + at);
                    const words2 high = read_transposed(tile + (read_v8 ^ (j % kCols << 6)) + at);
                    return words4{low[0], low[1], high[0], high[1]};
                };
                float w[16];
                words4 weights[2];
                const auto weigh = [&](int i) {
                    w[i] = __builtin_amdgcn_exp2f(s[i] * a.scale - shift);
                    sum += w[i];
                    if (i & 1) {
                        weights[i >> 3][(i & 7) >> 1] = T::pack(w[i - 1], w[i]);
                    }
                };
                words4 ahead[2] = {key_piece(0), key_piece(1)};
                words4 columns[2];
#pragma unroll
                for (int c = 0; c < kSteps; ++c) {
                    const words4 x = ahead[c & 1];
                    if (c + 2 < kSteps) {
                        ahead[c & 1] = key_piece(c + 2);
                    } else {
                        columns[c + 2 - kSteps] = column(c + 2 - kSteps);
                    }
                    n = T::mfma32(x, q[c], n);
#pragma unroll
                    for (int i = c * 12 / kSteps; i < (c + 1) * 12 / kSteps; ++i) {
                        weigh(i);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                float most = -INFINITY;
#pragma unroll
                for (int j = 0; j < 2 * kCols; ++j) {
                    const words4 x = columns[j & 1];
                    if (j + 2 < 2 * kCols) {
                        columns[j & 1] = column(j + 2);
                    }
                    o[j % kCols] = T::mfma32(x, weights[j / kCols], o[j % kCols]);
                    if (j < kCols) {
#pragma unroll
                        for (int i = 12 + j * 4 / kCols; i < 12 + (j + 1) * 4 / kCols; ++i) {
                            weigh(i);
                        }
                    }
                    beside(j);
#pragma unroll
                    for (int i = j * 8 / kCols; i < (j + 1) * 8 / kCols; ++i) {
                        most = fmaxf(most, n[i]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                most = over_halves_max(most);
                if (!whole) {
                    cut_scores(n, bits, left);
                    most = largest(n);
                }
                follow(most);
                s = n;
            };

            int32_t base = from << unit_shift;
            // Ids before rows, as in the loop: its first wait would otherwise be for the rows as well.
            const Ids first = ids_of(base);
            Ids ids = ids_of(base + kTile);
            uint64_t now = look(base, first);
            load_all(base);
            lds_barrier();     // the buffers' last use
            store_all(0);
            uint64_t next = look(base + kTile, ids);
            ids = ids_of(base + 2 * kTile);
            load_all(base + kTile);
            lds_barrier();
            int buffer = 0;
            f32x16 s = scores(s_data, 0);
            // Whether some row sees fewer keys of the tile at `base` than it holds.
            bool ragged = own && base + kTile > first_visible;
            if (ragged || static_cast<uint32_t>(now) != 0xffffffffu) {
                cut_scores(s, static_cast<uint32_t>(now), own ? visible - base : 32);
            }
            follow(largest(s));
#pragma unroll 1
            for (; base < keys; base += kTile, buffer ^= 2 * Tile<kDim>::kSize) {
                const char* const tile = s_data + buffer;
                const char* const other = s_data + (buffer ^ (2 * Tile<kDim>::kSize));
                if (ragged && any_not_finite(tile, hidden(lane))) {
                    // A key that only some rows see has weight 0 for the others, and 0 * infinity is not 0: the infinities
                    // and NaN are added to the rows that see them (a weight is positive), then cleared.
                    const int32_t left = visible - base;
                    const int my_half = hidden(half);
#pragma unroll 1
                    for (int key = 0; key < kTile; ++key) {
#pragma unroll
                        for (int c = 0; c < kCols; ++c) {
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                const words2 x = *reinterpret_cast<const words2*>(
                                    tile + Tile<kDim>::kSize + Tile<kDim>::place(key, c * 4 + (i >> 2)) + my_half * 8);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    o[c][i + e] += key < left ? T::unbounded(x[e >> 1] >> (16 * (e & 1))) : 0.0f;
                                }
                            }
                        }
                    }
                    lds_barrier();
#pragma unroll 1
                    for (int at = hidden(tid) * 16; at < Tile<kDim>::kSize; at += kWaves * 64 * 16) {
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
                const uint32_t bits = static_cast<uint32_t>(now >> 32);
                const int32_t left = own ? visible - base : kTile;
                now = next;
                next = look(base + 2 * kTile, ids);
                ids = ids_of(base + 3 * kTile);
                step_on(s, tile, 0, tile, 1, !ragged && bits == 0xffffffffu, bits, left - 32, [&](int j) {
                    // The next tile's rows leave their registers for the one after's.
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        if (i * kCols / kLoads == j) {
                            store(buffer ^ (2 * Tile<kDim>::kSize), i);
                        }
                        if (kCols + i * kCols / kLoads == j) {
                            load(base + 2 * kTile, i);
                        }
                    }
                });
                lds_barrier();      // the other buffer holds the next tile
                ragged = own && base + 2 * kTile > first_visible;
                step_on(s, tile, 1, other, 0, !ragged && static_cast<uint32_t>(now) == 0xffffffffu,
                        static_cast<uint32_t>(now), left - kTile + (own ? 0 : kTile), [](int) {});
                lds_barrier();      // nobody reads this buffer any more
            }
        }

        sum = over_halves_sum(sum);
        const int end_lane = hidden(threadIdx.x) & 63, end_half = end_lane >> 5;
        const int32_t end_row = g.row_begin + wave * 32 + (end_lane & 31);
        if (end_row < g.rows) {
            const Launch& last = fresh();
            const AttentionArgs& z = last.a;
            const Phase& p = last.p[which];
            const bool whole = p.direct != 0 && g.begin == 0 && g.end == g.units;
            constexpr int kRows = 32 * kWaves;
            if (whole) {
                const float inverse = sum == 0 ? 0.0f : 1.0f / sum;
                const int32_t token = z.share_div.div(end_row), head = (g.head - token) * z.share + end_row;
                char* const to = z.out + (g.q.first + token) * z.o_token + head * z.o_head;
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const int element = c * 32 + end_half * 4 + 2 * i;
                        if (element < z.dim) {
                            *reinterpret_cast<words2*>(to + element * 2) =
                                words2{T::pack(o[c][i] * inverse, o[c][i + 1] * inverse),
                                       T::pack(o[c][i + 2] * inverse, o[c][i + 3] * inverse)};
                        }
                    }
                }
                if (end_half == 0 && z.lse != nullptr) {
                    z.lse[(g.q.first + token) * z.l_token + head * z.l_head] =
                        sum == 0 ? -INFINITY : (top * z.scale - T::kShift + log2f(sum)) * kLn2;
                }
            } else if (static_cast<uint32_t>(g.slot) < static_cast<uint32_t>(p.slots)) {
                float* const part = p.parts + static_cast<int64_t>(g.slot) * kRows * (kDim + 2);
                const int inside = wave * 32 + (end_lane & 31);
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        // wide_place of the row and quad
                        reinterpret_cast<f32x4*>(part)[((wave * kCols + c) * 4 + (i >> 2)) * 64 + end_lane] =
                            f32x4{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]};
                    }
                }
                if (end_half == 0) {
                    part[kRows * kDim + inside] = top == -INFINITY ? top : top * z.scale;
                    part[kRows * kDim + kRows + inside] = sum;
                }
            }
        }
    });
}

}  // namespace wide
}  // namespace ekv
