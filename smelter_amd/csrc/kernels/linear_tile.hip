// smelter_amd/csrc/kernels/linear_tile.hip — the instantiations of the tile kernel (linear_tile.hpp)
#include "linear_tile.hpp"

template <int XK, int WK> static int lin_tile_shape(const LinearParams& p, int shape, bool dma, hipStream_t s) {
    if constexpr (XK != SM_MX4) if (!dma)
        return shape == 1 ? lin_tile<XK, WK, 16, 2, 4, 8, 4, false>(p, s) : shape == 2 ? lin_tile<XK, WK, 32, 2, 2, 2, 1, false>(p, s) : lin_tile<XK, WK, 32, 2, 2, 2, 2, false>(p, s);
    return shape == 1 ? lin_tile<XK, WK, 16, 2, 4, 8, 4, true>(p, s) : shape == 2 ? lin_tile<XK, WK, 32, 2, 2, 2, 1, true>(p, s) : lin_tile<XK, WK, 32, 2, 2, 2, 2, true>(p, s);
}

int lin_tile_launch(const LinearParams& p, int x_kind, int w_kind, int shape, bool dma, hipStream_t s) {
    if (x_kind == SM_MX4) return lin_tile_shape<SM_MX4, SM_MX4>(p, shape, dma, s);
    if (w_kind == SM_MX4) return x_kind == SM_F16 ? lin_tile_shape<SM_F16, SM_MX4>(p, shape, dma, s) : lin_tile_shape<SM_BF16, SM_MX4>(p, shape, dma, s);
    return x_kind == SM_F16 ? lin_tile_shape<SM_F16, SM_F16>(p, shape, dma, s) : lin_tile_shape<SM_BF16, SM_BF16>(p, shape, dma, s);
}

// Joins the runs of a split product, or the products of the parts of fp32 rows: y = act(sum of the runs, in their order, + bias).  One thread per four
// columns of a slot; the group of a slot (for its bias) is found in the offsets.  Bound by the reading of the sums and its own launch: 3 - 6 us.
__global__ void lin_join_kernel(LinearParams p) {
    const int quads = (p.N + 3) >> 2;
    const unsigned units = (unsigned)p.M * (unsigned)quads;                          // (below 2^31: lin_plan)
    const bool vec = !p.gated || p.N % 4 == 0;                                       // the up columns of a gated layer start at N
    for (unsigned u = blockIdx.x * blockDim.x + threadIdx.x; u < units; u += gridDim.x * blockDim.x) {
        const unsigned s = u / (unsigned)quads; const int n = (int)(u - s * quads) * 4;
        int e = 0;
        if (p.offsets) {                                                             // the last offset that is not behind s (32 of them one after the other: 12.2 us instead of 5.6)
            for (int b = p.E; e < b;) { const int mid = (e + b + 1) >> 1; if (lin_clamp(p.offsets[mid], p.M) <= s) e = mid; else b = mid - 1; }
            if (e == p.E || lin_clamp(p.offsets[e], p.M) > s || lin_clamp(p.offsets[e + 1], p.M) <= s) continue;
        }
        const int power = p.power ? p.power[s] : 0;
        if (power == LIN_MARKED) continue;
        const float apart = p.power ? 0x1p-11f : 1.f;                                // a part against the one before it
        floatx4 z[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        for (int h = 0; h <= p.gated; h++) {
            const int c = n + (h ? p.N : 0);
            const float* src = p.part + (p.parts ? (long long)p.parts : 1ll) * s * p.part_ld + c;
            const long long step = p.parts ? p.part_ld : p.M * p.part_ld;
            float scale = 1.f;
            if (vec) {
#pragma unroll 4
                for (int q = 0; q < p.splits; q++) { z[h] += *(const floatx4*)(src + q * step) * scale; scale *= apart; }
            } else {
                for (int q = 0; q < p.splits; q++) { for (int i = 0; i < 4; i++) if (n + i < p.N) z[h][i] += src[q * step + i] * scale; scale *= apart; }
            }
            if (p.parts) {
                // under an infinite weight a later part's sum may be 0 times infinity: an infinity of the first stands; a slot without a row of x is zero (of runs, the sums are already)
                const bool none = p.rows && (p.rows[s] < 0 || p.rows[s] >= p.T);
                for (int i = 0; i < 4; i++) { const float first = n + i < p.N ? src[i] : 0.f; z[h][i] = none ? 0.f : __builtin_fabsf(first) == __builtin_inff() ? first : ldexpf(z[h][i], power); }
            }
            if (p.bias) for (int i = 0; i < 4; i++) if (n + i < p.N) z[h][i] += p.bias[(long long)e * p.w_rows + c + i];
        }
        float v[4];
        for (int i = 0; i < 4; i++) v[i] = p.gated ? lin_silu(z[0][i]) * z[1][i] : lin_act(z[0][i], p.act, p.slope);
        const long long o = s * p.y_ld + n;
        if (p.y_vec && n + 4 <= p.N) lin_store4(p.y, o, v, p.y_type);
        else for (int i = 0; i < 4; i++) if (n + i < p.N) lin_store1(p.y, o + i, v[i], p.y_type);
    }
}

int lin_join_launch(const LinearParams& p, hipStream_t s) {
    const long long blocks = (p.M * ((p.N + 3) / 4) + 255) / 256, cap = (long long)SM_NUM_CU * 32;
    lin_join_kernel<<<dim3((unsigned)(blocks < cap ? blocks : cap)), 256, 0, s>>>(p);
    SM_LAUNCH_CHECK();
    return SM_OK;
}
