// Attention of queries to the paged K/V pool (gfx950): behind a prefix that a group of requests shares, and over the
// Top-K slots of a decode step.
//
//   o = sum_j softmax_j(scale q . k_j) v_j,   lse = log sum_j exp(scale q . k_j)
//
// over the keys that a query token sees. With the running largest score m, the sum l = sum exp(s_j - m) and the
// weighted values a = sum exp(s_j - m) v_j, two parts of the keys join as m = max(m1, m2),
// l = l1 e^(m1 - m) + l2 e^(m2 - m), a likewise, and o = a / l; statistics and sums are held in 32 bits.
#include "../../include/ekv_kernels.h"
#include "ekv_common.h"
#include "ekv_tensor_util.h"
#include "ekv_vec.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <cmath>

namespace ekv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Token offset o of page p of one KV head: k + p * page_stride + o * token_stride (bytes), V likewise.
struct Cache {
    const char* k;
    const char* v;
    int64_t page_stride, token_stride, head_stride;
    int64_t pages;      // page ids 1 .. pages - 1 (or zero_below ..) name pages
    int64_t page_size;
    int64_t zero_below;
};

struct Args {
    const char* query;
    int64_t q_token, q_head;      // bytes
    char* out;
    int64_t o_token, o_head;
    float* lse;
    int64_t l_token, l_head;      // elements
    Cache cache;
    const void* tables;           // [R, M] own pages of each request (or the slots of each query token)
    int64_t table_row, table_col;
    int32_t table64;
    int64_t requests, columns;
    IndexRef rows, lengths, query_starts;
    const void* prefix_tables;    // [G, P]
    int64_t prefix_row, prefix_col;
    int32_t prefix64;
    int64_t prefix_columns;
    IndexRef prefix_lengths, group_starts;
    int64_t tokens, batch, groups, heads, kv_heads, dim;
    float scale;                  // times log2 e
};

__device__ __forceinline__ float to_float(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_float(__hip_bfloat16& y, float x) { y = __float2bfloat16(x); }
__device__ __forceinline__ void from_float(__half& y, float x) { y = __float2half(x); }

// One wave per (query token, query head); each key is read by kLanes lanes of 8 elements, 64 / kLanes keys at a time.
template <typename T, int kLanes>
__global__ __launch_bounds__(kThreads) void attend_kernel(const Args a) {
    constexpr int kKeys = 64 / kLanes;
    const int lane = threadIdx.x & 63;
    const int64_t item = int64_t{blockIdx.x} * kWaves + (threadIdx.x >> 6);
    if (item >= a.tokens * a.heads) {
        return;
    }
    const int64_t token = item / a.heads, head = item % a.heads;
    const int64_t kv_head = head / (a.heads / a.kv_heads);
    const int part = lane % kLanes, sub = lane / kLanes;
    const bool live = part * 8 < a.dim;
    float q[8], acc[8] = {}, m = -INFINITY, l = 0;
    const T* q_at = reinterpret_cast<const T*>(a.query + token * a.q_token + head * a.q_head) + part * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        q[e] = live ? to_float(q_at[e]) : 0.0f;
    }
    // The batch row that the token belongs to, and its place there.
    int64_t b = token, at = 0, count = 1;
    if (a.query_starts.data != nullptr) {
        b = -1;
        for (int64_t i = 0; i < a.batch; ++i) {
            const int64_t begin = a.query_starts[i], end = a.query_starts[i + 1];
            if (begin <= token && token < end) {
                b = i, at = token - begin, count = end - begin;
                break;
            }
        }
    } else if (token >= a.batch) {
        b = -1;
    }
    int64_t group = -1;
    for (int64_t g = 0; g < a.groups && b >= 0; ++g) {
        const int64_t begin = a.group_starts.data != nullptr ? a.group_starts[g] : 0;
        const int64_t end = a.group_starts.data != nullptr ? a.group_starts[g + 1] : a.batch;
        if (begin <= b && b < end) {
            group = g;
            break;
        }
    }
    for (int side = 0; side < 2; ++side) {
        int64_t keys = 0, page_base = 0, page_col = 0;
        const void* table = nullptr;
        int32_t is64 = 0;
        if (side == 0 && group >= 0) {
            keys = min(a.prefix_lengths[group], a.prefix_columns * a.cache.page_size);
            table = a.prefix_tables, is64 = a.prefix64;
            page_base = group * a.prefix_row, page_col = a.prefix_col;
        } else if (side == 1 && b >= 0) {
            const int64_t row = a.rows.data != nullptr ? a.rows[b] : b;
            if (row >= 0 && row < a.requests) {
                const int64_t length = a.lengths.data != nullptr ? a.lengths[b] : a.columns;
                keys = min(a.lengths.data != nullptr ? length - count + at + 1 : length,
                           a.columns * a.cache.page_size);
                table = a.tables, is64 = a.table64;
                page_base = row * a.table_row, page_col = a.table_col;
            }
        }
        for (int64_t j0 = 0; j0 < keys; j0 += kKeys) {
            const int64_t j = j0 + sub;
            int64_t page = -1;
            if (j < keys) {
                const int64_t entry = page_base + j / a.cache.page_size * page_col;
                page = is64 ? static_cast<const int64_t*>(table)[entry] : static_cast<const int32_t*>(table)[entry];
            }
            const bool seen = page >= a.cache.zero_below && page < a.cache.pages;
            float k[8], v[8], s = 0;
            const int64_t offset = page * a.cache.page_stride + j % a.cache.page_size * a.cache.token_stride +
                                   kv_head * a.cache.head_stride + part * 16;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                k[e] = seen && live ? to_float(reinterpret_cast<const T*>(a.cache.k + offset)[e]) : 0.0f;
                v[e] = seen && live ? to_float(reinterpret_cast<const T*>(a.cache.v + offset)[e]) : 0.0f;
                s += q[e] * k[e];
            }
#pragma unroll
            for (int d = 1; d < kLanes; d <<= 1) {
                s += __shfl_xor(s, d);
            }
            s = seen ? s * a.scale : -INFINITY;
            const float top = fmaxf(m, s);
            const float safe = top == -INFINITY ? 0.0f : top;
            const float keep = exp2f(m - safe), p = exp2f(s - safe);
            m = top;
            l = l * keep + p;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                acc[e] = acc[e] * keep + p * v[e];
            }
        }
    }
#pragma unroll
    for (int d = kLanes; d < 64; d <<= 1) {
        const float other = __shfl_xor(m, d);
        const float top = fmaxf(m, other);
        const float safe = top == -INFINITY ? 0.0f : top;
        const float mine = exp2f(m - safe), theirs = exp2f(other - safe);
        l = l * mine + __shfl_xor(l, d) * theirs;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            acc[e] = acc[e] * mine + __shfl_xor(acc[e], d) * theirs;
        }
        m = top;
    }
    if (sub == 0 && live) {
        T* to = reinterpret_cast<T*>(a.out + token * a.o_token + head * a.o_head) + part * 8;
        const float inverse = l > 0 ? 1.0f / l : (l == 0 ? 0.0f : l);   // a NaN sum stays one
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            from_float(to[e], acc[e] * inverse);
        }
    }
    if (lane == 0 && a.lse != nullptr) {
        a.lse[token * a.l_token + head * a.l_head] = l == 0 ? -INFINITY : (m + log2f(l)) * kLn2;
    }
}

// ---------------------------------------------------------------- host

void need_aligned(int64_t value, const char* what) {
    if (value % 16 != 0) {
        throw std::invalid_argument(std::string(what) + " must be a multiple of 16 bytes");
    }
}

// A [tokens, heads, dim] tensor of 16-bit floats whose rows are dense and whose pieces of 8 are 16-byte aligned.
const ekv_tensor& need_rows(const ekv_tensor* p, const char* name) {
    const ekv_tensor& t = need(p, name);
    need_ndim(t, 3, name);
    if (t.dtype != EKV_BFLOAT16 && t.dtype != EKV_FLOAT16) {
        throw std::invalid_argument(std::string(name) + " must be bfloat16 or float16");
    }
    need_data(t, name);
    if (t.shape[2] > 1 && t.stride[2] != 1) {
        throw std::invalid_argument(std::string(name) + " must be dense in its last dimension");
    }
    if (numel(t) > 0) {
        need_aligned(reinterpret_cast<int64_t>(t.data), (std::string(name) + " address").c_str());
        need_aligned(t.shape[0] > 1 ? t.stride[0] * 2 : 0, (std::string(name) + " token stride").c_str());
        need_aligned(t.shape[1] > 1 ? t.stride[1] * 2 : 0, (std::string(name) + " head stride").c_str());
    }
    return t;
}

const ekv_tensor& need_list(const ekv_tensor* p, int64_t extent, const char* name) {
    const ekv_tensor& t = need(p, name);
    need_ndim(t, 1, name);
    need_index(t, name);
    need_dim(t, 0, extent, name);
    need_data(t, name);
    return t;
}

// Query, output, statistics and cache: what both entry points share.
Args common_args(const ekv_tensor* query_p, const ekv_planes* planes, int64_t layer, int64_t kv_heads,
                 int64_t page_size, double scale, const ekv_tensor* out_p, const ekv_tensor* lse_p) {
    const ekv_tensor& query = need_rows(query_p, "query");
    const ekv_tensor& out = need_rows(out_p, "output");
    for (int d = 0; d < 3; ++d) {
        need_dim(out, d, query.shape[d], "output");
    }
    if (out.dtype != query.dtype) {
        throw std::invalid_argument("output must have the query's type");
    }
    Args a{};
    a.tokens = query.shape[0], a.heads = query.shape[1], a.dim = query.shape[2];
    a.kv_heads = kv_heads;
    if (kv_heads < 1 || a.heads < 1 || a.heads % kv_heads != 0) {
        throw std::invalid_argument("kv_heads must divide the query's heads");
    }
    if (a.dim < 8 || a.dim > 256 || a.dim % 8 != 0) {
        throw std::invalid_argument("the head size must be a multiple of 8 from 8 to 256");
    }
    if (a.tokens > (int64_t{1} << 30) / a.heads) {
        throw std::invalid_argument("more than 2^30 query rows");
    }
    if (!std::isfinite(scale)) {
        throw std::invalid_argument("scale must be finite");
    }
    if (planes == nullptr) {
        throw std::invalid_argument("planes are required");
    }
    if (planes->kv != 2 || planes->layers < 0 || planes->rows < 0) {
        throw std::invalid_argument("planes must hold K and V (kv 2)");
    }
    if (layer < 0 || layer >= planes->layers) {
        throw std::invalid_argument("layer " + std::to_string(layer) + " outside the pool's " +
                                    std::to_string(planes->layers));
    }
    if (page_size < 1 || page_size > (int64_t{1} << 30)) {
        throw std::invalid_argument("page_size must be from 1 to 2^30");
    }
    const int64_t row = kv_heads * a.dim * 2;
    Cache& c = a.cache;
    if (planes->row_bytes == row) {                       // a plane row is a token
        c.token_stride = planes->row_stride;
        c.page_stride = planes->row_stride * page_size;
        c.pages = planes->rows / page_size;
    } else if (planes->row_bytes == row * page_size) {    // a plane row is a page
        c.token_stride = row;
        c.page_stride = planes->row_stride;
        c.pages = planes->rows;
    } else {
        throw std::invalid_argument("plane rows hold " + std::to_string(planes->row_bytes) + " bytes: neither a token's " +
                                    std::to_string(row) + " nor a page's " + std::to_string(row * page_size));
    }
    if (planes->base == nullptr && planes->rows > 0) {
        throw std::invalid_argument("null plane base");
    }
    c.head_stride = a.dim * 2;
    c.page_size = page_size;
    c.zero_below = 1;
    c.k = static_cast<const char*>(planes->base) + layer * planes->layer_stride;
    c.v = c.k + planes->kv_stride;
    need_aligned(reinterpret_cast<int64_t>(c.k), "plane address");
    need_aligned(planes->kv_stride, "kv stride");
    need_aligned(planes->row_stride, "plane row stride");
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
    a.scale = static_cast<float>(scale * 1.4426950408889634);
    return a;
}

template <typename T>
void launch_attend(const Args& a, hipStream_t stream) {
    const int64_t groups = (a.tokens * a.heads + kWaves - 1) / kWaves;
    const dim3 grid(static_cast<uint32_t>(groups)), block(kThreads);
    if (a.dim <= 64) {
        attend_kernel<T, 8><<<grid, block, 0, stream>>>(a);
    } else if (a.dim <= 128) {
        attend_kernel<T, 16><<<grid, block, 0, stream>>>(a);
    } else {
        attend_kernel<T, 32><<<grid, block, 0, stream>>>(a);
    }
}

int launch(const Args& a, int32_t dtype, void* stream) {
    if (a.tokens == 0) {
        return 0;
    }
    if (dtype == EKV_BFLOAT16) {
        launch_attend<__hip_bfloat16>(a, static_cast<hipStream_t>(stream));
    } else {
        launch_attend<__half>(a, static_cast<hipStream_t>(stream));
    }
    check_hip(hipGetLastError(), "launch attention");
    return 0;
}

void need_workspace(uint64_t needed, const void* workspace, uint64_t bytes) {
    if (bytes < needed) {
        throw std::invalid_argument("the attention needs " + std::to_string(needed) + " workspace bytes, got " +
                                    std::to_string(bytes));
    }
    if (needed > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)) {
        throw std::invalid_argument("the workspace must be a 256-byte aligned device buffer");
    }
}

uint64_t prefix_workspace(int64_t tokens, int64_t batch, int64_t groups, int64_t heads, int64_t kv_heads, int64_t dim,
                          int64_t max_query) {
    if (tokens < 0 || batch < 0 || groups < 0 || heads < 1 || kv_heads < 1 || dim < 1 || max_query < 1) {
        throw std::invalid_argument("attention sizes must be positive");
    }
    return 0;
}

uint64_t topk_workspace(int64_t tokens, int64_t lanes, int64_t heads, int64_t kv_heads, int64_t dim) {
    if (tokens < 0 || lanes < 0 || heads < 1 || kv_heads < 1 || dim < 1) {
        throw std::invalid_argument("attention sizes must be positive");
    }
    return 0;
}

int shared_prefix(const ekv_prefix_attention_args& s, void* workspace, uint64_t workspace_bytes, void* stream) {
    Args a = common_args(s.query, s.planes, s.layer, s.kv_heads, s.page_size, s.scale, s.output, s.lse);
    const auto need_table = [&](const ekv_tensor* p, const char* name) -> const ekv_tensor& {
        const ekv_tensor& t = need(p, name);
        need_ndim(t, 2, name);
        need_index(t, name);
        need_data(t, name);
        if (t.shape[1] > ((int64_t{1} << 30) - 1) / s.page_size) {
            throw std::invalid_argument(std::string(name) + " rows may cover at most 2^30 - 1 tokens");
        }
        return t;
    };
    const ekv_tensor& tables = need_table(s.block_tables, "block_tables");
    const ekv_tensor& lengths = need(s.lengths, "lengths");
    need_ndim(lengths, 1, "lengths");
    need_index(lengths, "lengths");
    need_data(lengths, "lengths");
    a.batch = lengths.shape[0];
    if (a.batch > (int64_t{1} << 24)) {
        throw std::invalid_argument("more than 2^24 batch rows");
    }
    a.lengths = index_ref(lengths, 0);
    a.tables = tables.data;
    a.table_row = tables.stride[0], a.table_col = tables.stride[1], a.table64 = tables.dtype == EKV_INT64;
    a.requests = tables.shape[0], a.columns = tables.shape[1];
    if (s.rows != nullptr) {
        a.rows = index_ref(need_list(s.rows, a.batch, "rows"), 0);
    }
    if (s.max_query < 1) {
        throw std::invalid_argument("max_query must be positive");
    }
    if (s.query_starts != nullptr) {
        a.query_starts = index_ref(need_list(s.query_starts, a.batch + 1, "query_starts"), 0);
    } else if (a.tokens != a.batch) {
        throw std::invalid_argument("without query_starts every batch row has one query token: got " +
                                    std::to_string(a.tokens) + " for " + std::to_string(a.batch) + " rows");
    }
    if ((s.prefix_tables == nullptr) != (s.prefix_lengths == nullptr)) {
        throw std::invalid_argument("prefix_tables and prefix_lengths are given together");
    }
    if (s.prefix_tables != nullptr) {
        const ekv_tensor& prefix = need_table(s.prefix_tables, "prefix_tables");
        a.groups = prefix.shape[0];
        a.prefix_tables = prefix.data;
        a.prefix_row = prefix.stride[0], a.prefix_col = prefix.stride[1], a.prefix64 = prefix.dtype == EKV_INT64;
        a.prefix_columns = prefix.shape[1];
        a.prefix_lengths = index_ref(need_list(s.prefix_lengths, a.groups, "prefix_lengths"), 0);
        if (s.group_starts != nullptr) {
            a.group_starts = index_ref(need_list(s.group_starts, a.groups + 1, "group_starts"), 0);
        } else if (a.groups > 1) {
            throw std::invalid_argument("more than one prefix needs group_starts");
        }
    } else if (s.group_starts != nullptr) {
        throw std::invalid_argument("group_starts without prefix_tables");
    }
    need_workspace(prefix_workspace(a.tokens, a.batch, a.groups, a.heads, a.kv_heads, a.dim, s.max_query), workspace,
                   workspace_bytes);
    return launch(a, s.query->dtype, stream);
}

int topk(const ekv_tensor* query, const ekv_planes* planes, int64_t layer, int64_t kv_heads, const ekv_tensor* slots_p,
         int64_t zero_below, double scale, const ekv_tensor* out, const ekv_tensor* lse, void* workspace,
         uint64_t workspace_bytes, void* stream) {
    Args a = common_args(query, planes, layer, kv_heads, 1, scale, out, lse);
    const ekv_tensor& slots = need(slots_p, "slots");
    need_ndim(slots, 2, "slots");
    need_index(slots, "slots");
    need_dim(slots, 0, a.tokens, "slots");
    need_data(slots, "slots");
    if (slots.shape[1] > (int64_t{1} << 30) - 1) {
        throw std::invalid_argument("more than 2^30 - 1 lanes");
    }
    if (zero_below < 0) {
        throw std::invalid_argument("zero_below must not be negative");
    }
    a.cache.zero_below = zero_below;
    a.batch = a.tokens;
    a.tables = slots.data;
    a.table_row = slots.stride[0], a.table_col = slots.stride[1], a.table64 = slots.dtype == EKV_INT64;
    a.requests = a.tokens, a.columns = slots.shape[1];
    need_workspace(topk_workspace(a.tokens, a.columns, a.heads, a.kv_heads, a.dim), workspace, workspace_bytes);
    return launch(a, query->dtype, stream);
}

}  // namespace
}  // namespace ekv

extern "C" uint64_t ekv_shared_prefix_workspace_bytes(int64_t tokens, int64_t batch, int64_t groups, int64_t heads,
                                                      int64_t kv_heads, int64_t head_dim, int64_t max_query) {
    return ekv::guarded(~uint64_t{0}, [&] {
        return ekv::prefix_workspace(tokens, batch, groups, heads, kv_heads, head_dim, max_query);
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
    return ekv::guarded(~uint64_t{0}, [&] { return ekv::topk_workspace(tokens, lanes, heads, kv_heads, head_dim); });
}

extern "C" int ekv_topk_attention(const ekv_tensor* query, const ekv_planes* planes, int64_t layer, int64_t kv_heads,
                                  const ekv_tensor* slots, int64_t zero_below, double scale, const ekv_tensor* output,
                                  const ekv_tensor* lse, void* workspace, uint64_t workspace_bytes, void* stream) {
    return ekv::guarded(-1, [&] {
        return ekv::topk(query, planes, layer, kv_heads, slots, zero_below, scale, output, lse, workspace,
                         workspace_bytes, stream);
    });
}
