// The launches of the attention kernel for many query rows by itself: prompt pieces (gfx950).
#include "ekv_attention_wide.h"

namespace ekv {
namespace {

template <typename T, int kDim, int kWaves>
__global__ __launch_bounds__(kWaves * 64, kDim <= 128 ? 2 : 1) void wide_kernel(const Launch) {
    __shared__ __align__(16) char s_data[wide::lds_bytes<kDim>()];
    __shared__ LineCells<kWaves, 255> s_line;
    wide::run<T, kDim, kWaves>(0, blockIdx.x, gridDim.x, false, 0, s_data, s_line);
}

template <typename T, int kDim>
void launch_dim(const Launch& l, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(l.p[0].workgroups));
    if (l.p[0].row_shift == 7) {
        wide_kernel<T, kDim, 4><<<grid, 256, 0, stream>>>(l);
    } else if constexpr (kDim <= 128) {
        wide_kernel<T, kDim, 8><<<grid, 512, 0, stream>>>(l);
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

void launch_wide(const Launch& l, int32_t dtype, void* stream) {
    if (dtype == EKV_BFLOAT16) {
        launch_type<Bf16>(l, static_cast<hipStream_t>(stream));
    } else {
        launch_type<F16>(l, static_cast<hipStream_t>(stream));
    }
}

}  // namespace ekv
