// smelter_amd/csrc/kernels/linear_deep.hip — the instantiations of the kernel for few tiles (linear_deep.hpp)
#include "linear_deep.hpp"

template <int XK, int WK> static int lin_deep_shape(const LinearParams& p, int shape, hipStream_t s) {
    if (shape == 2) return lin_deep_fits<XK, WK, 1, 4>(p) ? lin_deep<XK, WK, 1, 4>(p, s) : 1;
    return lin_deep_fits<XK, WK, 2, 4>(p) ? lin_deep<XK, WK, 2, 4>(p, s) : 1;
}

int lin_deep_launch(const LinearParams& p, int x_kind, int w_kind, int shape, hipStream_t s) {
    if (w_kind == SM_MX4) return x_kind == SM_F16 ? lin_deep_shape<SM_F16, SM_MX4>(p, shape, s) : lin_deep_shape<SM_BF16, SM_MX4>(p, shape, s);
    return x_kind == SM_F16 ? lin_deep_shape<SM_F16, SM_F16>(p, shape, s) : lin_deep_shape<SM_BF16, SM_BF16>(p, shape, s);
}
