// Attention of many query rows to the same keys: a large batch against its shared prefix, prompt pieces against prefix
// and own tokens (gfx950).
//
// Mathematics, per wave of 32 query rows and 32 keys: S^T = K Q^T by 32x32x16 matrix instructions (keys down, rows
// across: a lane holds 16 scores of one row, its other half-wave the other 16), running largest score and sum per row,
// P^T = exp(S^T - m) rounded once to 16 bits, O^T += V^T P^T. As in the kernel for few rows, P stays in the registers
// that the first product left it in, and the transposed LDS read gives V^T in the same order of keys.
//
// What bounds it: the matrix pipes, and the LDS that feeds them. A workgroup's waves share each tile of 64 keys: K and V
// of the next tile go from registers into the other of two LDS buffers, and the one after's rows are loaded, while a
// tile is worked on; one barrier a tile. At a head size of 128 a tile is 32 KB of LDS reads and 32 matrix instructions a
// wave.
#include "ekv_attention.h"
#include "ekv_mfma.h"

namespace ekv {
namespace {

constexpr int kTile = 64;   // keys of a tile

__device__ __align__(256) const uint32_t zero_row[128] = {};

template <int kDim>
struct Tile {
    static constexpr int kBytes = kDim <= 64 ? 128 : (kDim <= 128 ? 256 : 512);   // of a row in LDS
    static constexpr int kPieces = kDim / 8;
    static constexpr int kSize = kTile * kBytes;
    // The 16-byte pieces of a row are permuted by exclusive or so that 16 lanes with 16 keys and one piece (K) and the
    // four rows of 64 bytes that a transposed read takes at a time (V) each meet every bank once.
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

template <typename T, int kDim, int kWaves>
__global__ __launch_bounds__(kWaves * 64, kDim <= 128 ? 2 : 1) void wide_kernel(const AttentionArgs a, const Phase p) {
    constexpr int kSteps = kDim / 16;              // matrix steps of the first product
    constexpr int kCols = kDim / 32;               // 32-column pieces of the output
    constexpr int kRowThreads = Tile<kDim>::kBytes / 16;               // threads that load a key's row
    constexpr int kKeysAtOnce = kWaves * 64 / kRowThreads;
    constexpr int kLoads = kTile / kKeysAtOnce;    // 16-byte pieces of K, and of V, that a thread loads a tile
    static_assert(kLoads >= 1, "a tile has at least one piece for every thread");
    __shared__ __align__(16) char s_data[2][2][Tile<kDim>::kSize];     // [buffer][K, V]
    __shared__ LineCells<kWaves> s_line;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(tid >> 6));
    const int load_key = tid / kRowThreads, load_piece = tid % kRowThreads;
    const char* const zeros = reinterpret_cast<const char*>(zero_row);
    const int pieces = a.dim >> 3;

    for_segments(a, p, s_line, [&](const Segment& g) {
        const int32_t row = g.row_begin + wave * 32 + col;     // the lane's query row
        const int32_t token = a.share_div.div(row), head = (g.head - token) * a.share + row;
        words4 q[kSteps];
        {
            const char* at = a.query + (g.q.first + token) * a.q_token + head * a.q_head;
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                const int piece = c * 2 + half;
                q[c] = *reinterpret_cast<const words4*>(row < g.rows && piece < pieces ? at + piece * 16 : zeros);
            }
        }
        const int32_t visible = seen_by(g.q, token);
        const int32_t first_visible = seen_by(g.q, g.row_begin / a.share);
        const int32_t last_row = min(g.row_begin + 32 * kWaves, g.rows) - 1;
        const int32_t last_visible = seen_by(g.q, last_row / a.share);

        f32x16 o[kCols];
        float top = -INFINITY, sum = 0;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                o[c][i] = 0;
            }
        }

        const int32_t prefix_end = prefix_units(g.q, p);
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
            const int32_t keys = min(own ? last_visible : g.q.prefix, to << p.unit_shift);
            const char* const k_head = a.cache.k + static_cast<uint64_t>(a.cache.head_stride) * g.head +
                                       (load_piece < pieces ? load_piece : 0) * 16;

            // Page id of key base + lane, or 0xffffffff; every wave holds all of a tile's.
            const auto ids_of = [&](int32_t base) {
                const int32_t key = base + lane;
                const char* at = table + static_cast<uint64_t>(a.cache.page.div(key)) * step;
                at = key < keys ? at : zeros;
                const uint32_t low = *reinterpret_cast<const uint32_t*>(at);
                const uint32_t high = *reinterpret_cast<const uint32_t*>(at + wide);
                return key < keys && (wide == 0 || high == 0) ? low : 0xffffffffu;
            };
            words4 k[kLoads], v[kLoads];
            const auto fetch = [&](int32_t base, uint32_t ids) {
                const bool good = ids >= a.cache.zero_below && ids < a.cache.pages;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int32_t inside_tile = i * kKeysAtOnce + load_key;
                    const uint32_t id = __shfl(ids, inside_tile);
                    const int32_t key = base + inside_tile;
                    const bool live = id >= a.cache.zero_below && id < a.cache.pages;
                    const uint32_t inside = key - a.cache.page.div(key) * a.cache.page.divisor;
                    const uint64_t offset = static_cast<uint64_t>(id) * a.cache.page_stride +
                                            static_cast<uint64_t>(inside) * a.cache.token_stride;
                    k[i] = *reinterpret_cast<const words4*>(live ? k_head + offset : zeros);
                    v[i] = *reinterpret_cast<const words4*>(live ? k_head + offset + a.cache.kv_stride : zeros);
                }
                return __ballot(good);
            };
            const auto store = [&](int buffer) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int at = Tile<kDim>::place(i * kKeysAtOnce + load_key, load_piece);
                    // K past the head size meets zeros of q and must not be an infinity; V's columns are not stored.
                    const words4 kept = load_piece < pieces ? k[i] : words4{0, 0, 0, 0};
                    *reinterpret_cast<words4*>(&s_data[buffer][0][at]) = kept;
                    *reinterpret_cast<words4*>(&s_data[buffer][1][at]) = v[i];
                }
            };

            int32_t base = from << p.unit_shift;
            uint64_t now = fetch(base, ids_of(base));
            uint32_t ids = ids_of(base + kTile);
            __syncthreads();     // the buffers' last use
            store(0);
            uint64_t next = fetch(base + kTile, ids);
            ids = ids_of(base + 2 * kTile);
            __syncthreads();
            int buffer = 0;
#pragma unroll 1
            for (; base < keys; base += kTile, buffer ^= 1) {
                store(buffer ^ 1);
                const uint64_t seen = now;
                now = next;
                next = fetch(base + 2 * kTile, ids);
                ids = ids_of(base + 3 * kTile);
                const char* const k_tile = s_data[buffer][0];
                const char* const v_tile = s_data[buffer][1];
                f32x16 s[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[b][i] = 0;
                    }
#pragma unroll
                    for (int c = 0; c < kSteps; ++c) {
                        const words4 x =
                            *reinterpret_cast<const words4*>(k_tile + Tile<kDim>::place(b * 32 + col, c * 2 + half));
                        s[b] = T::mfma32(x, q[c], s[b]);
                    }
                }
                // Whether some row sees fewer keys of this tile than it holds.
                const bool ragged = own && base + kTile > first_visible;
                float most = -INFINITY;
                if (ragged || seen != ~uint64_t{0}) {
                    const int32_t left = own ? visible - base : kTile;
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint32_t bits = static_cast<uint32_t>(seen >> (32 * b));
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int key = half * 4 + (i & 3) + 8 * (i >> 2);
                            s[b][i] = ((bits >> key) & 1) != 0 && b * 32 + key < left ? s[b][i] * a.scale : -INFINITY;
                        }
                    }
                } else {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        s[b] *= a.scale;
                    }
                }
#pragma unroll
                for (int b = 0; b < 2; ++b) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        most = fmaxf(most, s[b][i]);
                    }
                }
                most = fmaxf(top, over_halves_max(most));
                const float safe = most == -INFINITY ? 0.0f : most;
                if (__ballot(most > top) != 0) {
                    const float keep = __builtin_amdgcn_exp2f(top - safe);
                    sum *= keep;
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        o[c] *= keep;
                    }
                    top = most;
                }
                const float shift = safe - T::kShift;
                words4 weights[4];                    // 16 keys each
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        w[j] = __builtin_amdgcn_exp2f(s[u >> 1][(u & 1) * 8 + j] - shift);
                        sum += w[j];
                    }
                    weights[u] =
                        words4{T::pack(w[0], w[1]), T::pack(w[2], w[3]), T::pack(w[4], w[5]), T::pack(w[6], w[7])};
                }
                // V^T of 16 keys and 32 columns: lane (half, 16-column piece, i) names row 4 half + i / 4 (+ 8).
                const auto column = [&](int u, int c) {
                    const int i = lane & 15, key = u * 16 + half * 4 + (i >> 2);
                    const int piece = c * 4 + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1), byte = (i & 1) * 8;
                    const words2 low = read_transposed(v_tile + Tile<kDim>::place(key, piece) + byte);
                    const words2 high = read_transposed(v_tile + Tile<kDim>::place(key + 8, piece) + byte);
                    return words4{low[0], low[1], high[0], high[1]};
                };
                bool spoiled = false;
                if (ragged) {
                    // A key that only some rows see has weight 0 for the others, and 0 * infinity is not 0.
#pragma unroll 1
                    for (int at = lane * 16; at < Tile<kDim>::kSize; at += 64 * 16) {
                        const words4 x = *reinterpret_cast<const words4*>(v_tile + at);
                        spoiled |= not_finite<T>(x[0]) || not_finite<T>(x[1]) || not_finite<T>(x[2]) ||
                                   not_finite<T>(x[3]);
                    }
                    spoiled = __ballot(spoiled) != 0;
                }
                if (!spoiled) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
#pragma unroll
                        for (int c = 0; c < kCols; ++c) {
                            o[c] = T::mfma32(column(u, c), weights[u], o[c]);
                        }
                    }
                } else {
                    // One query token at a time: its rows take the product with the values that it sees.
                    const int32_t last = min(g.row_begin + wave * 32 + 32, g.rows) - 1;
#pragma unroll 1
                    for (int32_t t = (g.row_begin + wave * 32) / a.share; t <= last / a.share; ++t) {
                        const int32_t left = seen_by(g.q, t) - base;
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
#pragma unroll
                            for (int c = 0; c < kCols; ++c) {
                                words4 x = column(u, c);
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const int key = u * 16 + half * 4 + (j & 3) + 8 * (j >> 2);
                                    x[j >> 1] &= key < left ? 0xffffffffu : ((j & 1) != 0 ? 0x0000ffffu : 0xffff0000u);
                                }
                                const f32x16 sums = T::mfma32(x, weights[u], o[c]);
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    o[c][i] = token == t ? sums[i] : o[c][i];
                                }
                            }
                        }
                    }
                }
                __syncthreads();
            }
        }

        sum = over_halves_sum(sum);
        if (row < g.rows) {
            const bool whole = p.direct != 0 && g.begin == 0 && g.end == g.units;
            constexpr int kRows = 32 * kWaves;
            if (whole) {
                const float inverse = sum == 0 ? 0.0f : 1.0f / sum;
                char* const to = a.out + (g.q.first + token) * a.o_token + head * a.o_head;
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const int element = c * 32 + half * 4 + 2 * i;
                        if (element < a.dim) {
                            *reinterpret_cast<words2*>(to + element * 2) =
                                words2{T::pack(o[c][i] * inverse, o[c][i + 1] * inverse),
                                       T::pack(o[c][i + 2] * inverse, o[c][i + 3] * inverse)};
                        }
                    }
                }
                if (half == 0 && a.lse != nullptr) {
                    a.lse[(g.q.first + token) * a.l_token + head * a.l_head] =
                        sum == 0 ? -INFINITY : (top - T::kShift + log2f(sum)) * kLn2;
                }
            } else if (g.slot < p.slots) {
                float* const part = p.parts + static_cast<int64_t>(g.slot) * kRows * (kDim + 2);
                const int inside = wave * 32 + col;
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        *reinterpret_cast<f32x4*>(part + inside * kDim + c * 32 + half * 4 + 2 * i) =
                            f32x4{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]};
                    }
                }
                if (half == 0) {
                    part[kRows * kDim + inside] = top;
                    part[kRows * kDim + kRows + inside] = sum;
                }
            }
        }
    });
}

template <typename T, int kDim>
void launch_dim(const AttentionArgs& a, const Phase& p, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(p.workgroups));
    if (p.row_shift == 7) {
        wide_kernel<T, kDim, 4><<<grid, 256, 0, stream>>>(a, p);
    } else {
        wide_kernel<T, kDim, 8><<<grid, 512, 0, stream>>>(a, p);
    }
    check_hip(hipGetLastError(), "launch attention");
}

template <typename T>
void launch_type(const AttentionArgs& a, const Phase& p, hipStream_t stream) {
    switch (p.dim_pad) {
        case 64: launch_dim<T, 64>(a, p, stream); break;
        case 96: launch_dim<T, 96>(a, p, stream); break;
        case 128: launch_dim<T, 128>(a, p, stream); break;
        default: launch_dim<T, 256>(a, p, stream); break;
    }
}

}  // namespace

void launch_wide(const AttentionArgs& a, const Phase& p, int32_t dtype, void* stream) {
    if (dtype == EKV_BFLOAT16) {
        launch_type<Bf16>(a, p, static_cast<hipStream_t>(stream));
    } else {
        launch_type<F16>(a, p, static_cast<hipStream_t>(stream));
    }
}

}  // namespace ekv
