// smelter_amd/csrc/kernels/linear_tile.hip — the instantiations of the tile kernel (linear_tile.hpp)
#include "linear_tile.hpp"

template <int XK, int WK> static int lin_tile_shape(const LinearParams& p, int shape, bool dma, hipStream_t s) {
    if constexpr (XK != SM_MX4) if (!dma) return lin_tile<XK, WK, 2, 2, 2, 2, false>(p, s);
    return shape ? lin_tile<XK, WK, 2, 4, 4, 2, true>(p, s) : lin_tile<XK, WK, 2, 2, 2, 2, true>(p, s);
}

int lin_tile_launch(const LinearParams& p, int x_kind, int w_kind, int shape, bool dma, hipStream_t s) {
    if (x_kind == SM_MX4) return lin_tile_shape<SM_MX4, SM_MX4>(p, shape, dma, s);
    if (w_kind == SM_MX4) return x_kind == SM_F16 ? lin_tile_shape<SM_F16, SM_MX4>(p, shape, dma, s) : lin_tile_shape<SM_BF16, SM_MX4>(p, shape, dma, s);
    return x_kind == SM_F16 ? lin_tile_shape<SM_F16, SM_F16>(p, shape, dma, s) : lin_tile_shape<SM_BF16, SM_BF16>(p, shape, dma, s);
}
