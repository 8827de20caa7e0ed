// smelter_amd/csrc/kernels/linear_stream.hpp — linear layers on FEW rows (decoding, small groups): the weights stream through the registers once, nothing is staged.
//
// A block owns 16 slots of one group and two groups of 16 weight rows (32 output columns, or 16 gated ones: gate rows and up rows); its waves split K and join their sums in LDS, in a fixed
// order.  Bound by the weights' bytes: a lane holds 32 consecutive k of one weight row (64 bytes of fp16, or one or two 16-byte MX4 blocks), so that a wave reads whole 128 / 256-byte pieces
// of 16 rows; which k a matrix instruction multiplies does not matter as long as both operands agree, so x is read in the same order (k = 32 (4 it + g) + 8 i for lane group g, step i) and no
// operand is re-arranged.  MX4 weights under 16-bit x become 16-bit values in the registers.  bf16: value times scale, exact.  fp16: the range of 2^-24 .. 65504 does not hold every scale, so
// the values are taken relative to the largest scale of their 256 (row, k) neighbours and the partial sum is multiplied by it in fp32 (a block 2^23 below that neighbour rounds, by less
// than the fp32 sum does).
#pragma once
#include "linear.hpp"

// 32 consecutive k of a row starting at block `b` (k = 32 b): 16-bit = four loads of eight, MX4 = one of 32 codes
template <int KIND> struct LinBlk { static constexpr int NV = KIND == SM_MX4 ? 1 : 4; intx4_t v[NV]; };
template <int KIND> __device__ __forceinline__ void lin_load_block(LinBlk<KIND>& f, const char* row, int b, int nb, int K) {
    if constexpr (KIND == SM_MX4) {
        f.v[0] = intx4_t{0, 0, 0, 0};
        if (b < nb) __builtin_memcpy(&f.v[0], row + 16ll * b, 16);
    } else {
        if (32 * b + 32 <= K) {
#pragma unroll
            for (int i = 0; i < 4; i++) __builtin_memcpy(&f.v[i], row + 64ll * b + 16 * i, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) f.v[i] = lin_load8(row, 32 * b + 8 * i, K);
        }
    }
}

template <int XK, int WK> __global__ void lin_stream_kernel(LinearParams p) {
    constexpr int NB = 2, BL = WK == SM_MX4 ? 2 : 1;                    // weight row groups; blocks of 32 k per lane and step
    extern __shared__ float part[];                                     // [waves][NB][16 slots][17]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const long long mt = blockIdx.x / p.n_tiles; const int nt = (int)(blockIdx.x - mt * p.n_tiles);
    const LinTile tile = lin_find_tile(p, 16, mt, false);
    if (tile.rows == 0) return;
    const int nb = (p.K + 31) >> 5;
    const int cols = p.gated ? 16 : 32, n0 = nt * cols;
    // operand rows of this lane; rows behind the end repeat the last one and are not stored
    long long xrow = tile.row0 + (r < tile.rows ? r : tile.rows - 1);
    if (p.rows) xrow = p.rows[xrow];
    const bool live = xrow >= 0 && xrow < p.T;                          // a row index outside x reads as a row of zeros
    if (!live) xrow = 0;
    const char* xr = p.x + xrow * p.x_ld; const unsigned char* xsr = p.xs + xrow * p.xs_ld;
    const char* wr[NB]; const unsigned char* wsr[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        int n = n0 + r + (p.gated ? 0 : 16 * b); if (n >= p.N) n = p.N - 1;
        const long long row = n + (p.gated ? (long long)b * p.N : 0);
        wr[b] = p.w + tile.e * p.w_es + row * p.w_ld;
        if constexpr (WK == SM_MX4) wsr[b] = p.ws + tile.e * p.ws_es + row * p.ws_ld;
    }
    floatx4 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) acc[b] = floatx4{0, 0, 0, 0};

    const int steps = (nb + 4 * BL - 1) / (4 * BL);
    for (int it = wave; it < steps; it += waves) {
        const int b0 = it * 4 * BL + g * BL;                            // this lane's first block
        LinBlk<WK> w[NB][BL]; int sc[NB][BL];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < BL; j++) {
                lin_load_block<WK>(w[b][j], wr[b], b0 + j, nb, p.K);
                sc[b][j] = 0;
                if constexpr (WK == SM_MX4) if (b0 + j < nb) sc[b][j] = wsr[b][b0 + j];
            }
        if constexpr (XK == SM_MX4) {
#pragma unroll
            for (int j = 0; j < BL; j++) {
                LinBlk<SM_MX4> x; int sx = 0;
                lin_load_block<SM_MX4>(x, xr, live ? b0 + j : nb, nb, p.K);
                if (live && b0 + j < nb) sx = xsr[b0 + j];
#pragma unroll
                for (int b = 0; b < NB; b++) acc[b] = lin_mma4(x.v[0], sx, w[b][j].v[0], sc[b][j], acc[b]);
            }
        } else {
            float mul[NB], rel[NB][BL];
            floatx4 sum[NB];
            if constexpr (WK == SM_MX4) {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    mul[b] = 1.f;
                    if constexpr (XK == SM_F16) {
                        int top = sc[b][0];
#pragma unroll
                        for (int j = 1; j < BL; j++) top = top > sc[b][j] ? top : sc[b][j];
                        int o = __shfl_xor(top, 16); top = top > o ? top : o;
                        o = __shfl_xor(top, 32); top = top > o ? top : o;
                        if (top < 1) top = 1;
                        mul[b] = mx4_scale(top);                        // >= 2^-126
#pragma unroll
                        for (int j = 0; j < BL; j++) { int d = sc[b][j] - top + 127; rel[b][j] = mx4_scale(sc[b][j] == 255 ? 255 : (d > 0 ? d : 0)); }
                    } else {
#pragma unroll
                        for (int j = 0; j < BL; j++) rel[b][j] = mx4_scale(sc[b][j]);
                    }
                }
            }
            constexpr bool OWN = WK == SM_MX4 && XK == SM_F16;          // partial sums of their own
#pragma unroll
            for (int b = 0; b < NB; b++) sum[b] = OWN ? floatx4{0, 0, 0, 0} : acc[b];
#pragma unroll
            for (int j = 0; j < BL; j++) {
                LinBlk<XK> x;
                lin_load_block<XK>(x, xr, b0 + j, nb, live ? p.K : 0);
#pragma unroll
                for (int i = 0; i < 4; i++) {
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        intx4_t v;
                        if constexpr (WK == SM_MX4) v = mx4_to16<XK>(w[b][j].v[0][i], rel[b][j]); else v = w[b][j].v[i];
                        sum[b] = lin_mma16<XK>(x.v[i], v, sum[b]);
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b++) acc[b] = OWN ? acc[b] + sum[b] * mul[b] : sum[b];
        }
    }
    // acc[b][i] = slot 4 g + i, weight row r of group b
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++) part[((wave * NB + b) * 16 + 4 * g + i) * 17 + r] = acc[b][i];
    __syncthreads();
    const float* bias = p.bias ? p.bias + (long long)tile.e * p.w_rows : nullptr;
    const int total = cols * tile.rows;
    for (int o = threadIdx.x; o < total; o += blockDim.x) {
        const int i = o / cols, c = o - i * cols, n = n0 + c;
        if (n >= p.N) continue;
        float v[2] = {0.f, 0.f};
        for (int h = 0; h < (p.gated ? 2 : 1); h++) {
            const int b = p.gated ? h : c >> 4;
            for (int q = 0; q < waves; q++) v[h] += part[((q * NB + b) * 16 + i) * 17 + (c & 15)];
            if (bias) v[h] += bias[n + (h ? p.N : 0)];
        }
        lin_store1(p.y, (tile.row0 + i) * p.y_ld + n, p.gated ? lin_silu(v[0]) * v[1] : lin_act(v[0], p.act, p.slope), p.y_type);
    }
}
