// Attention of few query rows to many keys: decode rows against their own pages, a small group against its prefix, a
// token against its Top-K slots (gfx950).
//
// Mathematics, per wave and 32 keys: S^T = K Q^T by 16x16x32 matrix instructions (keys down, 16 query rows across, so a
// lane holds 8 scores of one row), the running largest score and sum per row, P^T = exp(S^T - m) rounded once to 16 bits,
// O^T += V^T P^T. The lanes that hold a row's scores of keys 4g .. 4g + 3 and 16 + 4g .. are the lanes that feed them
// to the second product when its keys are taken in that order, so P never leaves its registers; V^T comes from a
// transposed read of LDS in the same order of keys.
//
// What bounds it: the K and V rows from HBM. Every wave reads its own keys (four waves a workgroup, each every
// fourth tile), K straight into the registers of the first product, V by way of LDS, with the next tile's rows in
// flight while a tile is worked on and the one after's page ids before them: 16 KB a wave in flight at a head size
// of 128. Each row of 16 * kTiles rows is held by every wave and joined at the end of an item in a fixed order.
#include "ekv_attention.h"
#include "ekv_mfma.h"

namespace ekv {
namespace {

constexpr int kKeys = 32;   // keys of a tile

// What a key that is not seen reads: weight 0 must meet a finite V.
__device__ __align__(256) const uint32_t zero_row[128] = {};

template <int kDim>
struct Rows {
    // LDS bytes of a V row, a power of two so that its 16-byte pieces can be permuted by exclusive or.
    static constexpr int kBytes = kDim <= 64 ? 128 : (kDim <= 128 ? 256 : 512);
    static __device__ __forceinline__ int place(int key, int piece) {
        // Rows are permuted so that 16 lanes with 16 keys and one piece meet 16 different 16-byte columns.
        const int swap = kBytes == 128 ? (key >> 1) & 7 : key & 15;
        return key * kBytes + ((piece ^ swap) << 4);
    }
};

template <int kDim, int kTiles>
constexpr int lds_bytes() {
    const int values = kAttentionWaves * kKeys * Rows<kDim>::kBytes;      // V of each wave's tile
    const int join = kAttentionWaves * 4 * kTiles * 64 * 16;              // four 16-column pieces of each wave's sums
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

// A tile of keys: where it lies, and the page id of each of the lane's two keys (l % 16 and 16 + l % 16 of the tile).
struct Pages {
    int32_t low[2], high[2];
};

// K and V rows of a tile, in the lane order of the first product: key l % 16 (+ 16), pieces l / 16 + 4 c.
template <int kSteps>
struct Held {
    words4 k[2][kSteps], v[2][kSteps];
    uint32_t seen;            // bit per key
};

template <typename T, int kDim, int kTiles>
__global__ __launch_bounds__(kAttentionThreads, kTiles == 1 && kDim <= 128 ? 2 : 1) void narrow_kernel(
    const AttentionArgs a, const Phase p) {
    constexpr int kSteps = kDim / 32;      // matrix steps of the first product
    constexpr int kCols = kDim / 16;       // 16-column pieces of the output
    __shared__ __align__(16) char s_data[lds_bytes<kDim, kTiles>()];
    __shared__ float s_max[kAttentionWaves][kTiles * 16], s_sum[kAttentionWaves][kTiles * 16];
    __shared__ LineCells s_line;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    char* const values = s_data + wave * (kKeys * Rows<kDim>::kBytes);
    const char* const zeros = reinterpret_cast<const char*>(zero_row);
    const int pieces = a.dim >> 3;

    for_segments(a, p, s_line, [&](const Segment& g) {
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
                const bool live = row < g.rows && piece < pieces;
                q[m][c] = *reinterpret_cast<const words4*>(live ? at + piece * 16 : zeros);
            }
            visible[m] = clamped(g.q.length - g.q.count + token + 1, 0, g.q.own);
        }
        const int32_t first_visible =
            __builtin_amdgcn_readfirstlane(clamped(g.q.length - g.q.count + g.row_begin / a.share + 1, 0, g.q.own));
        const int32_t prefix_tiles = (g.q.prefix + kKeys - 1) / kKeys;
        const bool prefix64 = a.prefix64, own64 = a.table64;

        const auto pages_of = [&](int32_t t) {
            Pages e;
            const bool own = t >= prefix_tiles;
            const int32_t base = (own ? t - prefix_tiles : t) * kKeys;
            const int32_t keys = t < g.end ? (own ? g.q.own : g.q.prefix) : 0;
            const bool wide = own ? own64 : prefix64;
            const char* table = static_cast<const char*>(own ? a.tables : a.prefix_tables);
            const int64_t start = own ? g.q.request * a.table_row : g.q.group * a.prefix_row;
            const int64_t step = own ? a.table_col : a.prefix_col;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int32_t key = base + h * 16 + col;
                const int64_t at = (start + a.cache.page.div(key) * step) * (wide ? 8 : 4);
                const char* from = key < keys ? table + at : zeros;
                e.low[h] = *reinterpret_cast<const int32_t*>(from);
                e.high[h] = *reinterpret_cast<const int32_t*>(from + (wide ? 4 : 0));
            }
            return e;
        };
        const auto rows_of = [&](int32_t t, const Pages& e) {
            Held<kSteps> d;
            const bool own = t >= prefix_tiles;
            const int32_t base = (own ? t - prefix_tiles : t) * kKeys;
            const int32_t keys = t < g.end ? (own ? g.q.own : g.q.prefix) : 0;
            const bool wide = own ? own64 : prefix64;
            d.seen = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int32_t key = base + h * 16 + col;
                const int32_t high = wide ? e.high[h] : e.low[h] >> 31;
                const int64_t page = static_cast<int64_t>(
                    (static_cast<uint64_t>(static_cast<uint32_t>(high)) << 32) | static_cast<uint32_t>(e.low[h]));
                const bool seen = key < keys && page >= a.cache.zero_below && page < a.cache.pages;
                const uint32_t inside = key - a.cache.page.div(key) * a.cache.page.divisor;
                const char* at = a.cache.k + page * a.cache.page_stride + inside * a.cache.token_stride +
                                 g.head * a.cache.head_stride;
#pragma unroll
                for (int c = 0; c < kSteps; ++c) {
                    const int piece = c * 4 + quad;
                    const bool live = seen && piece < pieces;
                    d.k[h][c] = *reinterpret_cast<const words4*>(live ? at + piece * 16 : zeros);
                    d.v[h][c] = *reinterpret_cast<const words4*>(live ? at + a.cache.kv_stride + piece * 16 : zeros);
                }
                d.seen |= (static_cast<uint32_t>(__ballot(seen)) & 0xffffu) << (16 * h);
            }
            return d;
        };

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
        int32_t t = g.begin + wave;
        Pages ahead = pages_of(t);
        Held<kSteps> next = rows_of(t, ahead);
        ahead = pages_of(t + kAttentionWaves);
        for (; t < g.end; t += kAttentionWaves) {
            const Held<kSteps> now = next;
            const Pages later = pages_of(t + 2 * kAttentionWaves);
            next = rows_of(t + kAttentionWaves, ahead);
            ahead = later;
            const bool own = t >= prefix_tiles;
            const int32_t base = (own ? t - prefix_tiles : t) * kKeys;
            // Whether some row sees fewer keys of this tile than it holds.
            const bool ragged = own && base + kKeys > first_visible;
            f32x4 s[kTiles][2];
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    s[m][h] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < kSteps; ++c) {
                        s[m][h] = T::mfma16(now.k[h][c], q[m][c], s[m][h]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int c = 0; c < kSteps; ++c) {
                    *reinterpret_cast<words4*>(values + Rows<kDim>::place(h * 16 + col, c * 4 + quad)) = now.v[h][c];
                }
            }
            words4 weights[kTiles];
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
                float x[8], most = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[j] = s[m][j >> 2][j & 3] * a.scale;
                }
                if (ragged || now.seen != 0xffffffffu) {
                    const int32_t left = own ? visible[m] - base : kKeys;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int key = (j >> 2) * 16 + quad * 4 + (j & 3);
                        x[j] = ((now.seen >> key) & 1) != 0 && key < left ? x[j] : -INFINITY;
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    most = fmaxf(most, x[j]);
                }
                most = fmaxf(top[m], over_groups_max(most));
                const float safe = most == -INFINITY ? 0.0f : most;
                if (__ballot(most > top[m]) != 0) {
                    const float keep = exp2f(top[m] - safe);
                    sum[m] *= keep;
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        o[m][c] *= keep;
                    }
                    top[m] = most;
                }
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = __builtin_amdgcn_exp2f(x[j] - safe + T::kShift);
                    sum[m] += w[j];
                }
                weights[m] = words4{T::pack(w[0], w[1]), T::pack(w[2], w[3]), T::pack(w[4], w[5]), T::pack(w[6], w[7])};
            }
            const auto column = [&](int c) {
                // Row quad * 4 + col / 4 of each 16 keys, the (col % 4)-th 8 bytes of the 32-byte column piece.
                const int key = quad * 4 + (col >> 2), piece = c * 2 + ((col & 3) >> 1), half = (col & 1) * 8;
                const words2 low = read_transposed(values + Rows<kDim>::place(key, piece) + half);
                const words2 high = read_transposed(values + Rows<kDim>::place(16 + key, piece) + half);
                return words4{low[0], low[1], high[0], high[1]};
            };
            bool spoiled = false;
            if (ragged) {
                // A key that only some rows see has weight 0 for the others, and 0 * infinity is not 0.
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int c = 0; c < kSteps; ++c) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            spoiled |= not_finite<T>(now.v[h][c][e]);
                        }
                    }
                }
                spoiled = __ballot(spoiled) != 0;
            }
            if (!spoiled) {
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    const words4 v = column(c);
#pragma unroll
                    for (int m = 0; m < kTiles; ++m) {
                        o[m][c] = T::mfma16(v, weights[m], o[m][c]);
                    }
                }
            } else {
                // One query token at a time: its rows take the product with the values that it sees.
                const int32_t last = min(g.row_begin + 16 * kTiles, g.rows) - 1;
                for (int32_t token = g.row_begin / a.share; token <= last / a.share; ++token) {
                    const int32_t left = clamped(g.q.length - g.q.count + token + 1, 0, g.q.own) - base;
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        words4 v = column(c);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int key = (j >> 2) * 16 + quad * 4 + (j & 3);
                            v[j >> 1] &= key < left ? 0xffffffffu : ((j & 1) != 0 ? 0x0000ffffu : 0xffff0000u);
                        }
#pragma unroll
                        for (int m = 0; m < kTiles; ++m) {
                            const f32x4 x = T::mfma16(v, weights[m], o[m][c]);
                            const int32_t row = g.row_begin + m * 16 + col;
                            o[m][c] = static_cast<int32_t>(a.share_div.div(row)) == token ? x : o[m][c];
                        }
                    }
                }
            }
        }

        // The waves' parts, joined in the order of the waves.
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            sum[m] = over_groups_sum(sum[m]);
            if (quad == 0) {
                s_max[wave][m * 16 + col] = top[m];
                s_sum[wave][m * 16 + col] = sum[m];
            }
        }
        __syncthreads();
        const bool whole = p.direct != 0 && g.begin == 0 && g.end == g.tiles;
        float* const part = p.parts + static_cast<int64_t>(g.slot) * p.row_tile * (p.dim_pad + 2);
        const bool room = g.slot < p.slots;
        float all_sum[kTiles];
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            float most = -INFINITY, total = 0;
#pragma unroll
            for (int w = 0; w < kAttentionWaves; ++w) {
                most = fmaxf(most, s_max[w][m * 16 + col]);
            }
            const float safe = most == -INFINITY ? 0.0f : most;
#pragma unroll
            for (int w = 0; w < kAttentionWaves; ++w) {
                total += s_sum[w][m * 16 + col] * exp2f(s_max[w][m * 16 + col] - safe);
            }
            const float mine = exp2f(top[m] - safe);
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                o[m][c] *= mine;
            }
            all_sum[m] = total;
            const int32_t row = g.row_begin + m * 16 + col;
            if (wave == 0 && quad == 0 && row < g.rows) {
                if (!whole) {
                    if (room) {
                        part[p.row_tile * p.dim_pad + m * 16 + col] = most;
                        part[p.row_tile * p.dim_pad + p.row_tile + m * 16 + col] = total;
                    }
                } else if (a.lse != nullptr) {
                    const int32_t place = a.share_div.div(row);
                    const int32_t token = g.q.first + place, head = (g.head - place) * a.share + row;
                    a.lse[token * a.l_token + head * a.l_head] =
                        total == 0 ? -INFINITY : (most - T::kShift + log2f(total)) * kLn2;
                }
            }
        }
        f32x4* const cells = reinterpret_cast<f32x4*>(s_data);   // [wave][column of the round][row tile][lane]
#pragma unroll
        for (int round = 0; round < (kCols + 3) / 4; ++round) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (round * 4 + c < kCols) {
#pragma unroll
                    for (int m = 0; m < kTiles; ++m) {
                        cells[((wave * 4 + c) * kTiles + m) * 64 + lane] = o[m][round * 4 + c];
                    }
                }
            }
            __syncthreads();
            const int piece = round * 4 + wave;
            if (piece < kCols) {
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
                    f32x4 x = cells[(wave * kTiles + m) * 64 + lane];
#pragma unroll
                    for (int w = 1; w < kAttentionWaves; ++w) {
                        x += cells[((w * 4 + wave) * kTiles + m) * 64 + lane];
                    }
                    const int32_t row = g.row_begin + m * 16 + col;
                    const int32_t element = piece * 16 + quad * 4;
                    if (row < g.rows) {
                        if (!whole) {
                            if (room) {
                                *reinterpret_cast<f32x4*>(part + (m * 16 + col) * p.dim_pad + element) = x;
                            }
                        } else if (element < a.dim) {
                            const float inverse = all_sum[m] == 0 ? 0.0f : 1.0f / all_sum[m];
                            const int32_t place = a.share_div.div(row);
                            const int32_t token = g.q.first + place, head = (g.head - place) * a.share + row;
                            *reinterpret_cast<words2*>(a.out + token * a.o_token + head * a.o_head + element * 2) =
                                words2{T::pack(x[0] * inverse, x[1] * inverse), T::pack(x[2] * inverse, x[3] * inverse)};
                        }
                    }
                }
            }
            __syncthreads();
        }
    });
}

template <typename T, int kDim>
void launch_dim(const AttentionArgs& a, const Phase& p, int tiles16, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(p.workgroups)), block(kAttentionThreads);
    if (tiles16 == 1) {
        narrow_kernel<T, kDim, 1><<<grid, block, 0, stream>>>(a, p);
    } else if (tiles16 == 2) {
        narrow_kernel<T, kDim, 2><<<grid, block, 0, stream>>>(a, p);
    } else if constexpr (kDim <= 128) {
        narrow_kernel<T, kDim, 4><<<grid, block, 0, stream>>>(a, p);
    }
    check_hip(hipGetLastError(), "launch attention");
}

template <typename T>
void launch_type(const AttentionArgs& a, const Phase& p, int tiles16, hipStream_t stream) {
    switch (p.dim_pad) {
        case 64: launch_dim<T, 64>(a, p, tiles16, stream); break;
        case 96: launch_dim<T, 96>(a, p, tiles16, stream); break;
        case 128: launch_dim<T, 128>(a, p, tiles16, stream); break;
        default: launch_dim<T, 256>(a, p, tiles16, stream); break;
    }
}

}  // namespace

void launch_narrow(const AttentionArgs& a, const Phase& p, int32_t dtype, int tiles16, void* stream) {
    if (dtype == EKV_BFLOAT16) {
        launch_type<Bf16>(a, p, tiles16, static_cast<hipStream_t>(stream));
    } else {
        launch_type<F16>(a, p, tiles16, static_cast<hipStream_t>(stream));
    }
}

}  // namespace ekv
