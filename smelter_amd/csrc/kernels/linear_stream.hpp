// smelter_amd/csrc/kernels/linear_stream.hpp — linear layers on FEW rows (decoding, small groups): the weights stream through the registers once, nothing is staged.
//
// A block owns 16 slots of one group and NB groups of 16 weight rows (16 NB output columns, or half as many gated ones: gate rows and up rows); its waves split K and join their sums in LDS, in a
// fixed order.  Bound by the weights' bytes (MX4 by MX4 reads them at 4.5 TB/s, 16-bit weights at 4.3, MX4 under a 16-bit x at 3.8: 4 rows of 262144 x 2048): a wave reads 128 or 256 bytes of each of
// its rows at once; which k a matrix instruction multiplies does not matter as long as both operands agree, so x is read in the same order and no operand is re-arranged.  What else goes through a
// CU's L1 is kept small beside the weights: the scales come as one dword per lane for 16 blocks and are handed to their lanes by a shuffle (byte loads cost 8 of 28 us of a 5-row layer of 16384 x 8192),
// lanes without a slot load no x, and where there are blocks enough a wave takes four groups of weight rows with the same x.
// MX4 weights under 16-bit x become 16-bit values in the registers.  bf16: value times scale, exact.  fp16: the range of 2^-24 .. 65504 does not hold every scale, so the values are taken
// relative to the largest scale of their row in these 512 k, exact where the scales are less than 2^36 apart, and the partial sum is multiplied by it in fp32; a wave that met others multiplies its
// share of K again as bf16 (lin_exact_blocks).
// fp32 x on fp16 weights (the rows that fp16 parts do not hold, linear.hip): the weights become fp32 values and the products are those of the fp32 matrix instruction, 1/16 of the fp16 rate.
#pragma once
#include "linear.hpp"

// 32 k of a row for a lane of group g.  ROW (16-bit x and weights): eight k of each of the blocks b .. b + 3, so that a row's four lanes read 64 bytes side by side (16 rows of 8192 x 8192: 31.1 us
// against 32.8 with a block for each); otherwise the lane's own block b: four loads of eight, or one of 32 MX4 codes.
template <int KIND> struct LinBlk { static constexpr int NV = KIND == SM_MX4 ? 1 : KIND == SM_F32 ? 8 : 4; intx4_t v[NV]; };
template <int KIND, bool ROW> __device__ __forceinline__ void lin_load_block(LinBlk<KIND>& f, const char* row, int b, int g, int nb, int K) {
    if constexpr (KIND == SM_F32) {                                     // the same k as of a 16-bit operand with ROW
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int k = 32 * (b + i) + 8 * g;
            if (k + 8 <= K) { __builtin_memcpy(&f.v[2 * i], row + 4ll * k, 16); __builtin_memcpy(&f.v[2 * i + 1], row + 4ll * k + 16, 16); }
            else {
#pragma unroll
                for (int q = 0; q < 8; q++) { int e = 0; if (k + q < K) __builtin_memcpy(&e, row + 4ll * (k + q), 4); f.v[2 * i + (q >> 2)][q & 3] = e; }
            }
        }
    } else if constexpr (ROW) {
        if (32 * b + 128 <= K) {
#pragma unroll
            for (int i = 0; i < 4; i++) __builtin_memcpy(&f.v[i], row + 64ll * (b + i) + 16 * g, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) f.v[i] = lin_load8(row, 32 * (b + i) + 8 * g, K);
        }
    } else if constexpr (KIND == SM_MX4) {
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

// four scale bytes of the blocks b .. b + 3 of a row, zero behind its end
__device__ __forceinline__ unsigned lin_load_scales4(const unsigned char* row, int b, int nb) {
    unsigned v = 0;
    if (b + 4 <= nb) __builtin_memcpy(&v, row + b, 4);
    else {
#pragma unroll
        for (int i = 0; i < 3; i++) if (b + i < nb) v |= (unsigned)row[b + i] << (8 * i);
    }
    return v;
}

template <int XK, int WK, int NB> __global__ __launch_bounds__(512) void lin_stream_kernel(LinearParams p) {
    constexpr bool MXW = WK == SM_MX4;
    constexpr int BL = MXW ? 2 : 1, U = MXW ? 2 : 1, CB = 4 * BL * U;  // blocks of 32 k per lane and step; steps of a chunk; blocks of a chunk
    extern __shared__ float part[];                                     // [waves][NB][16 slots][17]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const long long mt = blockIdx.x / (unsigned)p.n_tiles; const int nt = (int)(blockIdx.x - mt * p.n_tiles);
    const LinTile tile = lin_find_tile(p, 16, mt, false);
    if (tile.rows == 0) return;
    const int nb = (p.K + 31) >> 5;
    constexpr int G = NB / 2;                                           // groups of gate rows of a gated layer
    const int cols = p.gated ? 16 * G : 16 * NB, n0 = nt * cols;
    long long xrow = tile.row0 + (r < tile.rows ? r : 0);
    if (p.rows) xrow = p.rows[xrow];
    bool live = r < tile.rows;
    if constexpr (XK == SM_F32) {                                       // the marked rows only
        live = live && p.power[tile.row0 + r] == LIN_MARKED;
        if (!__any(live)) return;
    }
    const unsigned wanted = (unsigned)__ballot(live);
    live = live && xrow >= 0 && xrow < p.T;         // lanes without a slot, and row indices outside x: zeros
    if (!live) xrow = 0;
    const char* xr = p.x + xrow * p.x_ld; const unsigned char* xsr = p.xs + xrow * p.xs_ld;
    const int xk = live ? p.K : 0, xnb = live ? nb : 0;
    const char* wr[NB]; const unsigned char* wsr[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        int n = n0 + r + 16 * (p.gated ? b % G : b); if (n >= p.N) n = p.N - 1;
        const long long row = n + (p.gated && b >= G ? (long long)p.N : 0);
        wr[b] = p.w + tile.e * p.w_es + row * p.w_ld;
        wsr[b] = p.ws + tile.e * p.ws_es + row * p.ws_ld;
    }
    floatx4 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) acc[b] = floatx4{0, 0, 0, 0};

    int low = 255;                                                      // fp16 x on MX4: the smallest scale, relative to the largest of its row and chunk
    for (int c = wave * CB; c < nb; c += waves * CB) {
        // the weights of a chunk are asked for at once: a wave's share of K is short, what counts is how much of it is under way
        LinBlk<WK> w[U][NB][BL]; unsigned wsc[NB], xsc = 0;
#pragma unroll
        for (int b = 0; b < NB; b++) { wsc[b] = 0; if constexpr (MXW) wsc[b] = lin_load_scales4(wsr[b], c + 4 * g, nb); }
        if constexpr (XK == SM_MX4) xsc = lin_load_scales4(xsr, c + 4 * g, xnb);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < BL; j++) lin_load_block<WK, !MXW>(w[u][b][j], wr[b], MXW ? c + u * 4 * BL + g * BL + j : c, g, nb, p.K);
        // the scales of this lane's blocks c + 8 u + 2 g + {0, 1} lie in lane group 2 u + g / 2, bytes 2 (g & 1) + {0, 1}
        auto pair = [&](unsigned dw, int u) { return (unsigned)__shfl((int)dw, r + 16 * (2 * u + (g >> 1))) >> (16 * (g & 1)); };
        if constexpr (XK == SM_MX4) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const unsigned sx = pair(xsc, u);
                unsigned sw[NB];
#pragma unroll
                for (int b = 0; b < NB; b++) sw[b] = pair(wsc[b], u);
#pragma unroll
                for (int j = 0; j < BL; j++) {
                    LinBlk<SM_MX4> x;
                    lin_load_block<SM_MX4, false>(x, xr, c + u * 4 * BL + g * BL + j, g, xnb, p.K);
#pragma unroll
                    for (int b = 0; b < NB; b++) acc[b] = lin_mma4<0>(x.v[0], (int)(sx >> (8 * j)), w[u][b][j].v[0], (int)(sw[b] >> (8 * j)), acc[b]);
                }
            }
        } else if constexpr (XK == SM_F32) {
            static_assert(WK == SM_F16, "fp32 rows: fp16 weights (others take bf16 parts of them)");
            LinBlk<XK> x;
            lin_load_block<XK, true>(x, xr, c, g, nb, xk);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const float xe = __builtin_bit_cast(float, (int)x.v[2 * i + (q >> 2)][q & 3]);
#pragma unroll
                    for (int b = 0; b < NB; b++) acc[b] = lin_mma32(xe, (float)__builtin_bit_cast(half8_t, w[0][b][0].v[i])[q], acc[b]);
                }
        } else {
            constexpr bool OWN = MXW && XK == SM_F16;                   // sums of their own, multiplied by `mul`
            float mul[NB]; int top[NB]; floatx4 sum[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) {
                sum[b] = OWN ? floatx4{0, 0, 0, 0} : acc[b];
                if constexpr (OWN) {
                    int t = 14;
#pragma unroll
                    for (int i = 0; i < 4; i++) t = lin_top_of(t, wsc[b] >> (8 * i) & 255);
                    int o = __shfl_xor(t, 16); t = t > o ? t : o;
                    o = __shfl_xor(t, 32); top[b] = t > o ? t : o;
                    mul[b] = lin_top_scale(top[b]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                unsigned sw[NB];
                if constexpr (MXW) {
#pragma unroll
                    for (int b = 0; b < NB; b++) sw[b] = pair(wsc[b], u);
                }
#pragma unroll
                for (int j = 0; j < BL; j++) {
                    LinBlk<XK> x;
                    lin_load_block<XK, !MXW>(x, xr, MXW ? c + u * 4 * BL + g * BL + j : c, g, nb, xk);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        float rel = 0.f;
                        if constexpr (MXW) {
                            int byte = sw[b] >> (8 * j) & 255;
                            if constexpr (OWN) { byte = lin_relative(byte, top[b]); if (c + u * 4 * BL + g * BL + j < nb) low = low < byte ? low : byte; }
                            rel = mx4_scale(byte);
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            intx4_t v;
                            if constexpr (MXW) v = mx4_to16<XK>(w[u][b][j].v[0][i], rel); else v = w[u][b][j].v[i];
                            sum[b] = lin_mma16<XK>(x.v[i], v, sum[b]);
                        }
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b++) { if constexpr (OWN) acc[b] += sum[b] * mul[b]; else acc[b] = sum[b]; }
        }
    }
    if constexpr (MXW && XK == SM_F16) if (__any(low < 140 - LIN_REACH)) {   // blocks that fp16 does not hold beside the largest of their chunk: are they all zero?
        int far = 0;
        for (int c = wave * CB; c < nb; c += waves * CB)
#pragma unroll
            for (int b = 0; b < NB; b++) {
                int top = 14;
                for (int i = 0; i < CB && c + i < nb; i++) top = lin_top_of(top, wsr[b][c + i]);
                for (int i = g; i < CB && c + i < nb; i += 4)
                    if (lin_relative(wsr[b][c + i], top) < 140 - LIN_REACH) { intx4_t code; __builtin_memcpy(&code, wr[b] + 16ll * (c + i), 16); far |= (code[0] | code[1] | code[2] | code[3]) & 0x77777777; }
            }
        if (__any(far)) {
            const char* const xrow[1] = {xr}; const int xks[1] = {xk};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                floatx4 sum = {0, 0, 0, 0};
                for (int c = wave * CB; c < nb; c += waves * CB) {
                    floatx4 own = {0, 0, 0, 0};                         // (of these blocks: raised by itself)
                    lin_exact_blocks<16, 1>(wr[b], wsr[b], xrow, xks, c, c + CB < nb ? c + CB : nb, [&](int, intx4_t wf, intx4_t xf) { own = lin_mma16<SM_BF16>(xf, wf, own); },
                                            [&] { own = own * 0x1p64f * 0x1p64f; });
                    sum += own;
                }
                acc[b] = sum;
            }
        }
    }
    // acc[b][i] = slot 4 g + i, weight row r of group b; a slot without a row of x: zero, also under weights that are infinite or NaN
    const unsigned alive = (unsigned)__ballot(live) >> (4 * g);
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++) part[((wave * NB + b) * 16 + 4 * g + i) * 17 + r] = alive >> i & 1 ? acc[b][i] : 0.f;
    __syncthreads();
    const float* bias = p.bias ? p.bias + (long long)tile.e * p.w_rows : nullptr;
    const int total = cols * tile.rows;
    for (int o = threadIdx.x; o < total; o += blockDim.x) {
        const int i = o / cols, c = o - i * cols, n = n0 + c;
        if (n >= p.N || (XK == SM_F32 && !(wanted >> i & 1))) continue;
        float v[2] = {0.f, 0.f};
        for (int h = 0; h < (p.gated ? 2 : 1); h++) {
            const int b = (c >> 4) + h * G;
            for (int q = 0; q < waves; q++) v[h] += part[((q * NB + b) * 16 + i) * 17 + (c & 15)];
            if (bias) v[h] += bias[n + (h ? p.N : 0)];
        }
        lin_store1(p.y, (tile.row0 + i) * p.y_ld + n, p.gated ? lin_silu(v[0]) * v[1] : lin_act(v[0], p.act, p.slope), p.y_type);
    }
}
