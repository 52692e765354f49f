// The launches of the attention kernel for few query rows by itself: batches without a shared prefix, Top-K slots
// (gfx950).
#include "ekv_attention_narrow.h"

namespace ekv {
namespace {

template <typename T, int kDim, int kTiles>
__global__ __launch_bounds__(narrow::kWaves * 64, (narrow::groups_of<kDim, kTiles>())) void narrow_kernel(const Launch) {
    __shared__ __align__(16) char s_data[narrow::lds_bytes<kDim, kTiles>()];
    __shared__ __align__(16) char s_stats[narrow::stats_bytes<kTiles>()];
    __shared__ LineCells<narrow::kWaves, 255> s_line;
    narrow::run<T, kDim, kTiles>(0, blockIdx.x, gridDim.x, false, 0, s_data, s_stats, s_line);
}

template <typename T, int kDim>
void launch_dim(const Launch& l, int tiles16, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(l.p[0].workgroups)), block(narrow::kWaves * 64);
    if (tiles16 == 1) {
        narrow_kernel<T, kDim, 1><<<grid, block, 0, stream>>>(l);
    } else if (tiles16 == 2) {
        narrow_kernel<T, kDim, 2><<<grid, block, 0, stream>>>(l);
    } else if constexpr (kDim <= 128) {
        narrow_kernel<T, kDim, 4><<<grid, block, 0, stream>>>(l);
    }
    check_hip(hipGetLastError(), "launch attention");
}

template <typename T>
void launch_type(const Launch& l, int tiles16, hipStream_t stream) {
    switch (l.p[0].dim_pad) {
        case 64: launch_dim<T, 64>(l, tiles16, stream); break;
        case 96: launch_dim<T, 96>(l, tiles16, stream); break;
        case 128: launch_dim<T, 128>(l, tiles16, stream); break;
        default: launch_dim<T, 256>(l, tiles16, stream); break;
    }
}

}  // namespace

int narrow_groups(int tiles16, int32_t dim_pad) {
    return (tiles16 == 1 && dim_pad <= 128) || (tiles16 == 2 && dim_pad == 64) ? 2 : 1;
}

void launch_narrow(const Launch& l, int32_t dtype, int tiles16, void* stream) {
    if (dtype == EKV_BFLOAT16) {
        launch_type<Bf16>(l, tiles16, static_cast<hipStream_t>(stream));
    } else {
        launch_type<F16>(l, tiles16, static_cast<hipStream_t>(stream));
    }
}

}  // namespace ekv
