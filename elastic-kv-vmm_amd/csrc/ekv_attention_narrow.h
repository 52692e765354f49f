// Attention of few query rows to many keys: decode rows against their own pages, a small group against its prefix, a
// token against its Top-K slots (gfx950).
//
// Mathematics, per wave and 32 keys: S^T = K Q^T by 16x16x32 matrix instructions (keys down, 16 query rows across, so a
// lane holds 8 scores of one row), the running largest score and sum per row, P^T = exp(S^T - m) rounded once to 16 bits,
// O^T += V^T P^T. The lanes that hold a row's scores of keys 4g .. 4g + 3 and 16 + 4g .. are the lanes that feed them
// to the second product when its keys are taken in that order, so P never leaves its registers; V^T comes from a
// transposed read of LDS in the same order of keys.
//
// What bounds it: the K and V rows from HBM. Every wave reads its own keys (each every kWaves-th tile of the segment), K
// straight into the registers of the first product, V by way of LDS. A tile's registers are free once the first
// product and the LDS write have taken them, so the next tile's rows are in flight during the rest of a tile, and the
// page ids of the one after before them: 16 KB a wave at a head size of 128. Two tiles in flight at a head size of 64
// gained nothing (71 us against 69), nor did non-temporal loads or transposed reads ahead of the products. Each row of
// 16 * kTiles rows is held by every wave and joined at the end of an item in a fixed order.
//
// The weights are rounded once to the inputs' type, which the matrix instructions take: at most 2^-8 (bfloat16) or 2^-11
// (float16) of a weight, as much as K and V carry themselves. Held as a sum of two such numbers they would cost a second
// product per tile of V. The sums add the weights as they were before the rounding.
//
// Measured: a Top-K step of 128 tokens, 2048 slots each (225 thousand of 262 name a row), 2 KV heads of 128, bfloat16:
// 230 MB in 54.5 us where passes take four pools of 0.5 GB in turn, 12 us less on one pool, part of which is still in the
// last-level cache. A step of 4 tokens and 256 slots takes 8.5 us, the latency of slots, rows, join and store one after
// the other: the rows come at 4.2 TB/s with it and 5.0 without (a streaming copy reaches 6.5).
#pragma once

#include "ekv_attention.h"
#include "ekv_mfma.h"

namespace ekv {
namespace narrow {

constexpr int kKeys = 32;   // keys of a tile
constexpr int kWaves = 4;

template <int kDim>
struct Rows {
    // LDS bytes of a V row, a power of two so that its 16-byte pieces can be permuted by exclusive or.
    static constexpr int kBytes = kDim <= 64 ? 128 : (kDim <= 128 ? 256 : 512);
    static __device__ __forceinline__ int place(int key, int piece) {
        // The pieces of a row are permuted so that 16 lanes with 16 keys and one piece (the write) and the eight rows of
        // 32 bytes that a transposed read takes at a time each meet every bank once.
        const int swap = kBytes == 128 ? (((key >> 1) & 3) << 1) | ((key >> 3) & 1) : ((key & 7) << 1) | ((key >> 3) & 1);
        return key * kBytes + ((piece ^ swap) << 4);
    }
};

// Two workgroups share a compute unit where the row tile's registers leave room: one's start and end of an item overlap
// the other's reading.
template <int kDim, int kTiles>
constexpr int groups_of() {
    return (kTiles == 1 && kDim <= 128) || (kTiles == 2 && kDim == 64) ? 2 : 1;
}

template <int kDim, int kTiles>
constexpr int lds_bytes() {
    const int values = kWaves * kKeys * Rows<kDim>::kBytes;       // V of each wave's tile
    const int join = kWaves * (kDim / 16) * kTiles * 64 * 16;     // each wave's weighted values
    return values > join ? values : join;
}

__device__ __forceinline__ float over_groups_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float over_groups_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// One of the two sources of an item's keys.
struct Source {
    const char* table;        // its row of the page table
    uint32_t step;            // bytes between columns
    uint32_t wide;            // 4 for int64 ids: the high word's place
    int32_t keys;
};

// Page ids of the lane's two keys of a tile (l % 16 and 16 + l % 16), as words: int64 ids whose high word is not zero
// name no page.
struct Ids {
    uint32_t low[2], high[2];
};

template <int kTiles>
constexpr int stats_bytes() {
    return 2 * kWaves * kTiles * 16 * static_cast<int>(sizeof(float));
}

// Workgroup w's part of phase `which` of the launch. s_data: lds_bytes(), stats: stats_bytes() of LDS.
template <typename T, int kDim, int kTiles, int kChunk>
__device__ __forceinline__ void run(int which, uint32_t w, uint32_t workgroups, bool read, uint32_t total,
                                    char* s_data, char* stats, LineCells<kWaves, kChunk>& cells) {
    constexpr int kSteps = kDim / 32;      // matrix steps of the first product
    constexpr int kCols = kDim / 16;       // 16-column pieces of the output
    // Head sizes between kDim and the next smaller class end in one of the last steps.
    constexpr int kWholeSteps = kDim == 64 ? 0 : (kDim == 96 ? 2 : (kDim == 128 ? 3 : 4));
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    float (*const s_max)[kTiles * 16] = reinterpret_cast<float (*)[kTiles * 16]>(stats);
    float (*const s_sum)[kTiles * 16] = s_max + kWaves;
    char* const values = s_data + wave * (kKeys * Rows<kDim>::kBytes);
    const char* const zeros = reinterpret_cast<const char*>(zero_row);

    for_segments(which, w, workgroups, read, total, cells, [&](const Segment& g) {
        const int lane = hidden(threadIdx.x) & 63, col = lane & 15, quad = lane >> 4;
        const AttentionArgs& a = fresh().a;
        const int pieces = a.dim >> 3;
        const float slack = kSlack / fmaxf(a.scale, 1e-30f);     // in raw scores
        // Query rows: row col of each 16, elements 32 c + 8 quad .. + 7.
        words4 q[kTiles][kSteps];
        int32_t visible[kTiles];           // own keys that the lane's rows see
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            const int32_t row = g.row_begin + m * 16 + col;
            const int32_t token = a.share_div.div(row), head = (g.head - token) * a.share + row;
            const char* at = a.query + (g.q.first + token) * a.q_token + head * a.q_head;
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                const int piece = c * 4 + quad;
                const bool live = row < g.rows && (c < kWholeSteps || piece < pieces);
                q[m][c] = load_global<words4>(live ? at + piece * 16 : zeros);
                q[m][c] ^= a.flip;
            }
            visible[m] = seen_by(g.q, token);
        }
        const int32_t first_visible = seen_by(g.q, a.share_div.div(g.row_begin));

        f32x4 o[kTiles][kCols];
        float top[kTiles], sum[kTiles];
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            top[m] = -INFINITY, sum[m] = 0;
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                o[m][c] = f32x4{0, 0, 0, 0};
            }
        }

        const int32_t unit_shift = fresh().p[which].unit_shift;
        const int32_t prefix_end = (g.q.prefix + (1 << unit_shift) - 1) >> unit_shift;
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
            // Tiles [first, last) of this source; a wave takes every kWaves-th.
            const bool own = side == 1;
            const int32_t from = own ? max(g.begin - prefix_end, 0) : g.begin;
            const int32_t to = own ? g.end - prefix_end : min(g.end, prefix_end);
            if (to <= from) {
                continue;
            }
            Source src;
            src.table = own ? a.tables + g.q.request * a.table_row : a.prefix_tables + g.q.group * a.prefix_row;
            src.step = own ? a.table_col : a.prefix_col;
            src.wide = (own ? a.table64 : a.prefix64) != 0 ? 4 : 0;
            src.keys = min(own ? g.q.own : g.q.prefix, to << unit_shift);
            const char* const k_head = a.cache.k + static_cast<uint64_t>(a.cache.head_stride) * g.head + quad * 16;
            const char* const v_head = k_head + a.cache.kv_stride;

            const Cache cache = a.cache;
            const auto ids_of = [&](int32_t base) {
                Ids e;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int32_t key = base + h * 16 + col;
                    const char* at = src.table + static_cast<uint64_t>(cache.page.div(key)) * src.step;
                    at = key < src.keys ? at : zeros;
                    e.low[h] = load_global<uint32_t>(at);
                    e.high[h] = load_global<uint32_t>(at + src.wide);
                }
                return e;
            };
            words4 k[2][kSteps], v[2][kSteps];
            uint32_t seen;                    // bit per key of the tile
            const auto fetch = [&](int32_t base, const Ids& e) {
                seen = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int32_t key = base + h * 16 + col;
                    const uint32_t id = e.low[h];
                    const bool good = key < src.keys && id >= cache.zero_below && id < cache.pages &&
                                      (src.wide == 0 || e.high[h] == 0);
                    const uint32_t inside = key - cache.page.div(key) * cache.page.divisor;
                    const uint64_t offset = static_cast<uint64_t>(id) * cache.page_stride +
                                            static_cast<uint64_t>(inside) * cache.token_stride;
                    const char* k_at = k_head + offset;
                    const char* v_at = v_head + offset;
                    k_at = good ? k_at : zeros;
                    v_at = good ? v_at : zeros;
#pragma unroll
                    for (int c = 0; c < kSteps; ++c) {
                        // Past the head size: any piece of the row; K meets zeros of q once it is cleared, V's columns
                        // are not stored.
                        const int piece = c < kWholeSteps || c * 4 + quad < pieces ? c * 64 : -quad * 16;
                        k[h][c] = load_global<words4>(k_at + (good || c < kWholeSteps ? piece : 0));
                        v[h][c] = load_global<words4>(v_at + (good || c < kWholeSteps ? piece : 0));
                    }
                    seen |= (static_cast<uint32_t>(__ballot(good)) & 0xffffu) << (16 * h);
                }
            };

            constexpr int kStride = kWaves * kKeys;
            const int32_t start = (from << unit_shift) + wave * kKeys;
            const Ids first = ids_of(start);
            Ids ids = ids_of(start + kStride);
            fetch(start, first);
            const auto tile = [&](int32_t base) {
                const Ids later = ids_of(base + 2 * kStride);
                const uint32_t now = seen;
                // Whether some row sees fewer keys of this tile than it holds.
                const bool ragged = own && base + kKeys > first_visible;
                f32x4 s[kTiles][2];
                if (kWholeSteps < kSteps && a.dim != kDim) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int c = kWholeSteps; c < kSteps; ++c) {
                            k[h][c] = c * 4 + quad < pieces ? k[h][c] : words4{0, 0, 0, 0};
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        s[m][h] = f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int c = 0; c < kSteps; ++c) {
                            s[m][h] = T::mfma16(k[h][c], q[m][c], s[m][h]);
                        }
                    }
                }
                bool spoiled = false;
                if (ragged) {
                    rarely();
                    // A key that only some rows see has weight 0 for the others, and 0 * infinity is not 0.
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int c = 0; c < kSteps; ++c) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                spoiled |= not_finite<T>(v[h][c][e]);
                            }
                        }
                    }
                    spoiled = __ballot(spoiled) != 0;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int c = 0; c < kSteps; ++c) {
                        *reinterpret_cast<words4*>(values + Rows<kDim>::place(h * 16 + col, c * 4 + quad)) = v[h][c];
                    }
                }
                fetch(base + kStride, ids);
                ids = later;
                words4 weights[kTiles];
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
                    float x[8], most = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        x[j] = s[m][j >> 2][j & 3];
                    }
                    if (ragged || now != 0xffffffffu) {
                        rarely();
                        const int32_t left = own ? visible[m] - base : kKeys;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int key = (j >> 2) * 16 + quad * 4 + (j & 3);
                            x[j] = ((now >> key) & 1) != 0 && key < left ? x[j] : -INFINITY;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        most = fmaxf(most, x[j]);
                    }
                    most = over_groups_max(most);
                    // The reference score follows the largest only when that has passed it by 2^kSlack: until then the
                    // weights are larger than 1, which their type holds, and nothing has to be scaled again.
                    if (__ballot(most > top[m] + slack) != 0) {
                        const float to = fmaxf(top[m], most);
                        const float keep = to == top[m] ? 1.0f : __builtin_amdgcn_exp2f((top[m] - to) * a.scale);
                        sum[m] *= keep;
#pragma unroll
                        for (int c = 0; c < kCols; ++c) {
                            o[m][c] *= keep;
                        }
                        top[m] = to;
                    }
                    const float shift = (top[m] == -INFINITY ? 0.0f : top[m] * a.scale) - T::kShift;
                    float w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        w[j] = __builtin_amdgcn_exp2f(x[j] * a.scale - shift);
                        sum[m] += w[j];
                    }
                    weights[m] =
                        words4{T::pack(w[0], w[1]), T::pack(w[2], w[3]), T::pack(w[4], w[5]), T::pack(w[6], w[7])};
                }
                const auto column = [&](int c) {
                    // Row quad * 4 + col / 4 of each 16 keys, the (col % 4)-th 8 bytes of the 32-byte column piece.
                    const int key = quad * 4 + (col >> 2), piece = c * 2 + ((col & 3) >> 1), half = (col & 1) * 8;
                    const words2 low = read_transposed(values + Rows<kDim>::place(key, piece) + half);
                    const words2 high = read_transposed(values + Rows<kDim>::place(16 + key, piece) + half);
                    return words4{low[0], low[1], high[0], high[1]};
                };
                if (spoiled) {
                    // A key that only some rows see has weight 0 for the others, and 0 * infinity is not 0: the infinities
                    // and NaN are added to the rows that see them (a weight is positive), then cleared.
                    const int my_quad = hidden(quad);
#pragma unroll 1
                    for (int key = 0; key < kKeys; ++key) {
#pragma unroll
                        for (int c = 0; c < kCols; ++c) {
                            words2* const at = reinterpret_cast<words2*>(
                                values + Rows<kDim>::place(key, c * 2 + (my_quad >> 1)) + (my_quad & 1) * 8);
                            const words2 x = *at;
#pragma unroll
                            for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    o[m][c][e] +=
                                        key < visible[m] - base ? T::unbounded(x[e >> 1] >> (16 * (e & 1))) : 0.0f;
                                }
                            }
                            *at = words2{bounded<T>(x[0]), bounded<T>(x[1])};
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    const words4 column_c = column(c);
#pragma unroll
                    for (int m = 0; m < kTiles; ++m) {
                        o[m][c] = T::mfma16(column_c, weights[m], o[m][c]);
                    }
                }
            };
#pragma unroll 1
            for (int32_t base = start; base < src.keys; base += kStride) {
                tile(base);
            }
        }

        // The waves' parts, joined in the order of the waves: each wave scales its values to the largest score of all,
        // then sums its columns of everybody's.
        const int end_lane = hidden(threadIdx.x) & 63, end_col = end_lane & 15, end_quad = end_lane >> 4;
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            sum[m] = over_groups_sum(sum[m]);
            top[m] = top[m] == -INFINITY ? top[m] : top[m] * a.scale;
            if (end_quad == 0) {
                s_max[wave][m * 16 + end_col] = top[m];
                s_sum[wave][m * 16 + end_col] = sum[m];
            }
        }
        lds_barrier();
        const Launch& last = fresh();
        const AttentionArgs& z = last.a;
        const Phase& p = last.p[which];
        const bool whole = p.direct != 0 && g.begin == 0 && g.end == g.units;
        const int32_t row_tile = 16 * kTiles;
        float* const part = p.parts + static_cast<int64_t>(g.slot) * row_tile * (kDim + 2);
        const bool room = static_cast<uint32_t>(g.slot) < static_cast<uint32_t>(p.slots);
        f32x4* const joined = reinterpret_cast<f32x4*>(s_data);   // [wave][column][row tile][end_lane]
        float factor[kTiles];
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            float most = -INFINITY, total = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                most = fmaxf(most, s_max[w][m * 16 + end_col]);
            }
            const float safe = most == -INFINITY ? 0.0f : most;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                total += s_sum[w][m * 16 + end_col] * __builtin_amdgcn_exp2f(s_max[w][m * 16 + end_col] - safe);
            }
            const float mine = __builtin_amdgcn_exp2f(top[m] - safe);
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                joined[((wave * kCols + c) * kTiles + m) * 64 + end_lane] = o[m][c] * mine;
            }
            factor[m] = !whole ? 1.0f : (total == 0 ? 0.0f : 1.0f / total);
            const int32_t row = g.row_begin + m * 16 + end_col;
            if (wave == 0 && end_quad == 0 && row < g.rows) {
                if (!whole) {
                    if (room) {
                        part[row_tile * kDim + m * 16 + end_col] = most;
                        part[row_tile * kDim + row_tile + m * 16 + end_col] = total;
                    }
                } else if (z.lse != nullptr) {
                    const int32_t token = z.share_div.div(row);
                    z.lse[(g.q.first + token) * z.l_token + ((g.head - token) * z.share + row) * z.l_head] =
                        total == 0 ? -INFINITY : (most - T::kShift + log2f(total)) * kLn2;
                }
            }
        }
        lds_barrier();
#pragma unroll
        for (int c = wave; c < kCols; c += kWaves) {
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
                f32x4 x = joined[(c * kTiles + m) * 64 + end_lane];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) {
                    x += joined[((w * kCols + c) * kTiles + m) * 64 + end_lane];
                }
                x *= factor[m];
                const int32_t row = g.row_begin + m * 16 + end_col;
                const int32_t element = c * 16 + end_quad * 4;
                if (row < g.rows) {
                    if (!whole) {
                        if (room) {
                            // narrow_place of the row and quad
                            reinterpret_cast<f32x4*>(part)[(c * kTiles + m) * 64 + end_lane] = x;
                        }
                    } else if (element < z.dim) {
                        const int32_t token = z.share_div.div(row), head = (g.head - token) * z.share + row;
                        *reinterpret_cast<words2*>(z.out + (g.q.first + token) * z.o_token + head * z.o_head +
                                                   element * 2) = words2{T::pack(x[0], x[1]), T::pack(x[2], x[3])};
                    }
                }
            }
        }
        lds_barrier();
    });
}

}  // namespace narrow
}  // namespace ekv
