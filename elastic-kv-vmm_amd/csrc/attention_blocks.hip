// The launches of the attention kernel for few query rows over lists of blocks (gfx950).
//
// What bounds it: the reading. 128 tokens' 32 blocks of 64, 2 KV heads of 128, 0.27 GB, take 59 us, 4.5 TB/s, and 5 for
// the merge. (Accesses of whole rows and K by way of LDS, as the selection reads its keys: 58, with the registers of the
// larger tiles spilled.) Four tokens' 4 blocks of 128 take 11 and 4.
#include "ekv_attention_narrow.h"

namespace ekv {
namespace {

template <typename T, int kDim, int kTiles>
__global__ __launch_bounds__(narrow::kWaves * 64, (narrow::groups_of<kDim, kTiles>())) void blocks_kernel(const Launch) {
    __shared__ __align__(16) char s_data[narrow::lds_bytes<kDim, kTiles>()];
    __shared__ __align__(16) char s_stats[narrow::stats_bytes<kTiles>()];
    __shared__ LineCells<narrow::kWaves, 255> s_line;
    narrow::run<T, kDim, kTiles, true>(0, blockIdx.x, gridDim.x, false, 0, s_data, s_stats, s_line);
}

template <typename T, int kDim>
void launch_dim(const Launch& l, int tiles16, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(l.p[0].workgroups)), block(narrow::kWaves * 64);
    if constexpr (kDim <= 128) {
        switch (tiles16) {
            case 1: blocks_kernel<T, kDim, 1><<<grid, block, 0, stream>>>(l); break;
            case 2: blocks_kernel<T, kDim, 2><<<grid, block, 0, stream>>>(l); break;
            default: blocks_kernel<T, kDim, 4><<<grid, block, 0, stream>>>(l); break;
        }
    } else {
        blocks_kernel<T, kDim, 1><<<grid, block, 0, stream>>>(l);
    }
    check_hip(hipGetLastError(), "launch block attention");
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

void launch_blocks(const Launch& l, int32_t dtype, int tiles16, void* stream) {
    if (dtype == EKV_BFLOAT16) {
        launch_type<Bf16>(l, tiles16, static_cast<hipStream_t>(stream));
    } else {
        launch_type<F16>(l, tiles16, static_cast<hipStream_t>(stream));
    }
}

}  // namespace ekv
