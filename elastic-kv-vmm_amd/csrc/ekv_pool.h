// Host-side checks that the operators over the paged pool share: rows of 16-bit floats, lists of indexes, where a
// token's row of a plane lies, and whether two tensors may share memory.
#pragma once

#include "ekv_fastdiv.h"
#include "ekv_tensor_util.h"

#include <algorithm>
#include <array>
#include <cstdlib>
#include <numeric>
#include <utility>

namespace ekv {

inline void need_aligned(int64_t value, const char* what) {
    if (value % 16 != 0) {
        throw std::invalid_argument(std::string(what) + " must be a multiple of 16 bytes");
    }
}

// A [tokens, heads, dim] tensor of 16-bit floats whose rows are dense and whose pieces of 8 are 16-byte aligned.
inline const ekv_tensor& need_rows(const ekv_tensor* p, const char* name) {
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

inline const ekv_tensor& need_list(const ekv_tensor* p, int64_t extent, const char* name) {
    const ekv_tensor& t = need(p, name);
    need_ndim(t, 1, name);
    need_index(t, name);
    need_dim(t, 0, extent, name);
    need_data(t, name);
    return t;
}

// Bytes between the columns of a table of page ids.
inline uint32_t column_step(const ekv_tensor& t, const char* name, int dim = 1) {
    const int64_t step = t.shape[dim] > 1 ? t.stride[dim] * itemsize(t.dtype) : 0;
    if (step < 0 || step > 0x7fffffff) {
        throw std::invalid_argument(std::string(name) + ": columns more than 2 GiB apart");
    }
    return static_cast<uint32_t>(step);
}

// Where token `offset` of page `page` lies in a plane of one layer: at + page * page_stride + offset * token_stride.
struct PlanePages {
    char* at = nullptr;
    int64_t kv_stride = 0, page_stride = 0, token_stride = 0, pages = 0;
};

// The pages of layer `layer` of planes whose rows hold a token (`row` bytes) or a whole page of them.
inline PlanePages plane_pages(const ekv_planes* planes, int64_t layer, int64_t row, int64_t page_size, int64_t kv) {
    if (planes == nullptr) {
        throw std::invalid_argument("planes are required");
    }
    if (planes->kv != kv || planes->layers < 0 || planes->rows < 0) {
        throw std::invalid_argument(kv == 2 ? "planes must hold K and V (kv 2)"
                                            : "planes must hold one plane a layer (kv 1)");
    }
    if (layer < 0 || layer >= planes->layers) {
        throw std::invalid_argument("layer " + std::to_string(layer) + " outside the pool's " +
                                    std::to_string(planes->layers));
    }
    if (page_size < 1 || page_size > (int64_t{1} << 30)) {
        throw std::invalid_argument("page_size must be from 1 to 2^30");
    }
    PlanePages p;
    constexpr int64_t kMostStride = 0xffffffff;
    if (planes->row_stride < 0 || planes->row_stride > kMostStride) {
        throw std::invalid_argument("the plane row stride must be below 4 GiB");
    }
    if (planes->row_bytes == row) {                       // a plane row is a token
        p.token_stride = planes->row_stride;
        p.page_stride = planes->row_stride * page_size;
        p.pages = planes->rows / page_size;
    } else if (planes->row_bytes == row * page_size) {    // a plane row is a page
        p.token_stride = row;
        p.page_stride = planes->row_stride;
        p.pages = planes->rows;
    } else {
        throw std::invalid_argument("plane rows hold " + std::to_string(planes->row_bytes) + " bytes: neither a token's " +
                                    std::to_string(row) + " nor a page's " + std::to_string(row * page_size));
    }
    if (planes->base == nullptr && planes->rows > 0) {
        throw std::invalid_argument("null plane base");
    }
    if (p.page_stride > kMostStride || p.pages > 0x7fffffff) {
        throw std::invalid_argument("a page must lie within 4 GiB, and a plane hold fewer than 2^31 pages");
    }
    p.at = static_cast<char*>(planes->base) + layer * planes->layer_stride;
    p.kv_stride = planes->kv_stride;
    need_aligned(reinterpret_cast<int64_t>(p.at), "plane address");
    if (kv > 1) {
        need_aligned(planes->kv_stride, "kv stride");
    }
    need_aligned(planes->row_stride, "plane row stride");
    return p;
}

// The bytes of a strided tensor: runs of `run` bytes that begin at multiples of `step` from `begin`.
struct Extent {
    int64_t begin = 0, end = 0, step = 0, run = 0;

    Extent() = default;

    explicit Extent(const ekv_tensor* t) {
        if (t == nullptr || numel(*t) == 0) {
            return;
        }
        const int64_t item = itemsize(t->dtype);
        begin = reinterpret_cast<int64_t>(t->data);
        end = begin + item;
        run = item;
        // Innermost dimensions that lie side by side are one run.
        int dim = t->ndim - 1;
        for (; dim >= 0; --dim) {
            if (t->shape[dim] > 1) {
                if (t->stride[dim] * item != run) {
                    break;
                }
                run *= t->shape[dim];
                end += (t->shape[dim] - 1) * t->stride[dim] * item;
            }
        }
        for (; dim >= 0; --dim) {
            if (t->shape[dim] > 1) {
                const int64_t apart = t->stride[dim] * item, reach = (t->shape[dim] - 1) * apart;
                step = std::gcd(step, apart);
                begin += std::min<int64_t>(reach, 0);
                end += std::max<int64_t>(reach, 0);
            }
        }
    }

    Extent(const void* data, uint64_t bytes) {
        if (bytes > 0) {
            begin = reinterpret_cast<int64_t>(data);
            run = static_cast<int64_t>(bytes);
            end = begin + run;
        }
    }

    // Plane `kv` of a layer.
    Extent(const PlanePages& p, const ekv_planes& planes, int64_t kv) {
        if (planes.rows > 0) {
            begin = reinterpret_cast<int64_t>(p.at) + kv * planes.kv_stride;
            end = begin + (planes.rows - 1) * planes.row_stride + planes.row_bytes;
            step = planes.row_stride;
            run = planes.row_bytes;
        }
    }

    // Whether the two may share a byte: runs of both lie at whole multiples of the steps' greatest common divisor from
    // each other, so that tensors that lie in one another, as slices of a fused projection, are told apart.
    bool meets(const Extent& other) const {
        if (run == 0 || other.run == 0 || begin >= other.end || other.begin >= end) {
            return false;
        }
        const int64_t common = std::gcd(step, other.step);
        if (common == 0) {
            return true;
        }
        const int64_t apart = ((other.begin - begin) % common + common) % common;
        return apart < run || common - apart < other.run;
    }
};

inline void need_apart(const Extent& a, const char* name, const Extent& b, const char* other) {
    if (a.meets(b)) {
        throw std::invalid_argument(std::string(name) + " must not share memory with " + other);
    }
}

// An output whose elements are all different: every dimension steps over the whole of those with smaller strides.
inline void need_distinct(const ekv_tensor& t, const char* name) {
    std::array<std::pair<int64_t, int64_t>, 4> dims;      // stride, extent
    int count = 0;
    for (int i = 0; i < t.ndim; ++i) {
        if (t.shape[i] > 1) {
            dims[count++] = {std::abs(t.stride[i]), t.shape[i]};
        }
    }
    std::sort(dims.begin(), dims.begin() + count);
    int64_t reach = 0;
    for (int i = 0; i < count && numel(t) > 0; ++i) {
        if (dims[i].first <= reach) {
            throw std::invalid_argument(std::string(name) + " must not repeat its elements");
        }
        reach += (dims[i].second - 1) * dims[i].first;
    }
}

// Rows of a plane that are written: no two share a byte.
inline void need_distinct_rows(const ekv_planes& planes) {
    if (planes.rows > 1 && planes.row_stride < planes.row_bytes) {
        throw std::invalid_argument("plane rows must not overlap");
    }
}

// Whether two tensors are the same elements.
inline bool same_view(const ekv_tensor& a, const ekv_tensor& b) {
    if (a.data != b.data || a.dtype != b.dtype || a.ndim != b.ndim) {
        return false;
    }
    for (int i = 0; i < a.ndim; ++i) {
        if (a.shape[i] != b.shape[i] || (a.shape[i] > 1 && a.stride[i] != b.stride[i])) {
            return false;
        }
    }
    return true;
}

}  // namespace ekv
