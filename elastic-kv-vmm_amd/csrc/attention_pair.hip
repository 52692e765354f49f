// Attention of a batch behind shared prefixes in one launch: own tokens and prefixes are two lines of work, and the
// workgroups are shared between them by what the lines cost (gfx950).
//
// Reading own tokens is bound by HBM, the product with a prefix by the matrix pipes once a group has enough rows. The
// first workgroups of the grid work on prefixes, the others on own tokens; the first and the second half of the grid are
// dealt to the compute units in turn, so that as long as both have work most units hold one of each. Both phases in
// every workgroup, one after the other, took 67 us where this takes 52 (with the merge; 32 requests of 32 heads, 8 KV
// heads of 128, 8192 tokens of prefix and up to 1024 own), 148 where it takes 109 (128 requests of 16 heads, 2 KV heads,
// 32768 and up to 4096): 112 MB in 43 us of this kernel, 338 MB in 101 to 111.
//
// At a head size of 128 the kernel for many rows has 25 vector registers more than two workgroups a compute unit leave
// it and keeps them in scratch (104 bytes a lane); at 256 it is 53 to 86.
#include "ekv_attention_narrow.h"
#include "ekv_attention_wide.h"

namespace ekv {
namespace {

constexpr int kWaves = 4;
static_assert(kWaves == narrow::kWaves, "one workgroup runs both");

template <int kDim>
constexpr int data_bytes() {
    return wide::lds_bytes<kDim>() > narrow::lds_bytes<kDim, 1>() ? wide::lds_bytes<kDim>() : narrow::lds_bytes<kDim, 1>();
}

// kFew: own tokens of at most 16 rows.
template <typename T, int kDim, bool kFew>
__global__ __launch_bounds__(kWaves * 64, kDim <= 128 ? 2 : 1) void pair_kernel(const Launch) {
    __shared__ __align__(16) char s_data[data_bytes<kDim>()];
    __shared__ __align__(16) char s_stats[narrow::stats_bytes<1>()];
    __shared__ LineCells<kWaves, 128> s_line[2];
    uint32_t totals[2];
    line_totals(totals, s_line);
    const Launch& l = fresh();
    const uint32_t share = prefix_workgroups(l.p[0], l.p[1], totals[0], totals[1]), b = blockIdx.x;
    if (kFew && b >= share) {
        narrow::run<T, kDim, 1>(0, on_die(b - share, gridDim.x - share), gridDim.x - share, true, totals[0], s_data,
                                s_stats, s_line[0]);
    } else {
        const int which = b < share ? 1 : 0;
        wide::run<T, kDim, kWaves>(which, which == 1 ? b : b - share, which == 1 ? share : gridDim.x - share, true,
                                   totals[which], s_data, s_line[which]);
    }
}

template <typename T, int kDim>
void launch_dim(const Launch& l, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(l.p[0].workgroups));
    if (l.p[0].row_shift == 4) {
        pair_kernel<T, kDim, true><<<grid, kWaves * 64, 0, stream>>>(l);
    } else {
        pair_kernel<T, kDim, false><<<grid, kWaves * 64, 0, stream>>>(l);
    }
    check_hip(hipGetLastError(), "launch attention");
}

template <typename T>
void launch_type(const Launch& l, hipStream_t stream) {
    switch (l.p[0].dim_pad) {
        case 64: launch_dim<T, 64>(l, stream); break;
        case 96: launch_dim<T, 96>(l, stream); break;
        case 128: launch_dim<T, 128>(l, stream); break;
        default: launch_dim<T, 256>(l, stream); break;
    }
}

}  // namespace

void launch_pair(const Launch& l, int32_t dtype, void* stream) {
    if (dtype == EKV_BFLOAT16) {
        launch_type<Bf16>(l, static_cast<hipStream_t>(stream));
    } else {
        launch_type<F16>(l, static_cast<hipStream_t>(stream));
    }
}

}  // namespace ekv
