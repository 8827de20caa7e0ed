// smelter_amd/csrc/kernels/linear_tile.hpp — linear layers on MANY rows: tiles of BN weight rows x BM slots through LDS, 128 bytes of K at a time.
//
// Both operands lie in LDS as rows of 128 bytes (64 16-bit elements, or 8 MX4 blocks = 256 elements), filled by the LDS-DMA without passing a register.  16-byte chunk c of row r sits at place
// c ^ (r & 7), for fragments of 32 rows at c ^ (r & 7) ^ (r >> 4 & 1): the sixteen lanes that a 16-byte LDS read serves together (0 - 3, 12 - 15, 20 - 23, 24 - 27 and their like) then touch all
// banks.  Without the second term 1000 x 4096 x 4096 in bfloat16 takes 50 us instead of 47; fragments of 16 rows with neighbouring chunks to a lane instead (their scales then lie together by
// themselves) make 42 % of the LDS cycles conflicts, 3 % of the time of 8192^3 in MX4.
// The weights are the first operand of the matrix instruction: a lane then holds four consecutive columns of one slot, which it stores together.  A product of 16-bit fragments and one of MX4
// fragments read the same bytes in the same order, so both kinds share the kernel; the MX4 one adds the scale bytes.  MX4 weights under a 16-bit x become 16-bit values on their way into LDS.
#pragma once
#include "linear.hpp"

// 16 bytes per lane from base + off -> lds + 16 * lane (base and lds wave-uniform); completion: s_waitcnt vmcnt
__device__ __forceinline__ void lin_dma16(const char* base, unsigned off, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(off), "s"(base), "s"(lds));
}
__device__ __forceinline__ unsigned lin_lds_addr(const void* p) { return (unsigned)(size_t)(const __attribute__((address_space(3))) void*)p; }
__device__ __forceinline__ void lin_arrive() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Which tile (and which run of K) this block has: consecutive tiles stay on one XCD (blocks are dealt to the 8 XCDs in turn), in squares of up to 8 row tiles, so that an XCD's L2 holds what its
// CUs read together.  The number of row tiles is known on the device only; blocks to spare get an empty tile.
// HALVES (a tile to a CU): where the last round of an XCD's tiles fills at most half of its CUs, two blocks take the halves of each of these tiles.
template <bool HALVES> __device__ __forceinline__ LinTile lin_pick_tile(const LinearParams& p, int BM, int* split, int* nt) {
    LinTile none; none.rows = 0;
    *split = p.splits > 1 ? (int)(blockIdx.x % (unsigned)p.splits) : 0;
    const LinTile all = lin_find_tile(p, BM, 0, true);
    const long long total = all.total * p.n_tiles;
    const long long b = p.splits > 1 ? blockIdx.x / (unsigned)p.splits : blockIdx.x, q = total >> 3;
    const int xcd = (int)(b & 7), rem = (int)(total & 7);
    const long long mine = q + (xcd < rem ? 1 : 0);                                 // tiles of this XCD
    long long at = b >> 3; int half = -1;
    if constexpr (HALVES) {
        const int over = (int)(mine % (SM_NUM_CU / 8));
        if (over <= SM_NUM_CU / 16 && at >= mine - over) { const int j = (int)(at - (mine - over)); half = j & 1; at = mine - over + (j >> 1); }
    }
    if (at >= mine) return none;
    const long long id = xcd * q + (xcd < rem ? xcd : rem) + at;
    const long long band = id / (8ll * p.n_tiles);
    const int in = (int)(id - band * 8 * p.n_tiles), high = (int)(all.total - band * 8 < 8 ? all.total - band * 8 : 8);
    *nt = in / high;
    LinTile tile = lin_find_tile(p, BM, band * 8 + in - *nt * high, false);
    if (HALVES && half >= 0) {
        if (half) { tile.row0 += BM / 2; tile.rows = tile.rows > BM / 2 ? tile.rows - BM / 2 : 0; }
        else if (tile.rows > BM / 2) tile.rows = BM / 2;
    }
    return tile;
}
// weight row of tile row j: gated tiles alternate 16 gate rows and their 16 up rows
__device__ __forceinline__ long long lin_weight_row(const LinearParams& p, int n0, int j) {
    int n = p.gated ? n0 + ((j >> 5) << 4) + (j & 15) : n0 + j;
    if (n >= p.N) n = p.N - 1;
    return n + (p.gated && (j & 16) ? (long long)p.N : 0);
}
// row of x of tile slot j (behind the tile's end: of its last slot), -1: outside x
__device__ __forceinline__ long long lin_slot_row(const LinearParams& p, const LinTile& tile, int j) {
    long long s = tile.row0 + (j < tile.rows ? j : tile.rows - 1);
    if (p.rows) { s = p.rows[s]; if (s < 0 || s >= p.T) s = -1; }
    return s;
}

// Epilogue of the tile kernels: acc[a][b][i] = tile row FR (wn FN + a) + 8 (i / 4) + 4 g + i % 4 of the weights, slot FR (wm FM + b) + r: quads of four consecutive columns of a slot, quad j of a
// lane at column CW j + 4 g of its wave; gate and up row of a column lie in the same lane.  SCALED: wmul[row] = the factor of a weight row.
template <int FR, int FN, int FM> struct LinQuads {
    static constexpr int Q = FR * FR / 256, N = FN * Q, CW = 256 / FR, UP = 16 / CW;   // quads of a fragment, of a wave; columns from one to the next; quads from a gate row to its up row
};
template <int FR, int FN, int FM, bool SCALED, int J, class AccT> __device__ __forceinline__ floatx4 lin_quad(const AccT (&acc)[FN][FM], int b, const float* wmul) {
    constexpr int Q = LinQuads<FR, FN, FM>::Q, q = J % Q;
    const AccT& c = acc[J / Q][b];
    floatx4 v = {c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]};
    if constexpr (SCALED) v *= *(const floatx4*)(wmul + LinQuads<FR, FN, FM>::CW * J);
    return v;
}

// The sums of a run of K, in the order of the weight rows; lin_join_kernel adds them.
template <int FR, int FN, int FM, bool SCALED, class AccT>
__device__ __forceinline__ void lin_finish_split(const LinearParams& p, const LinTile& tile, int split, int n0, int row0, const AccT (&acc)[FN][FM], const int (&slot)[FM], const float* wmul) {
    typedef LinQuads<FR, FN, FM> L;
    sm_static_for<0, L::N>([&](auto index) {
        constexpr int j = decltype(index)::value;
        const int row = row0 + L::CW * j, n = p.gated ? n0 + ((row >> 5) << 4) + (row & 15) : n0 + row;
#pragma unroll
        for (int b = 0; b < FM; b++) {
            const floatx4 v = lin_quad<FR, FN, FM, SCALED, j>(acc, b, wmul);
            if (slot[b] >= tile.rows || n >= p.N) continue;
            float* dst = p.part + ((long long)split * p.M + tile.row0 + slot[b]) * p.part_ld + n + (p.gated && (row & 16) ? p.N : 0);
            if (n + 4 <= p.N && (!p.gated || p.N % 4 == 0)) *(floatx4*)dst = v;
            else {
#pragma unroll
                for (int i = 0; i < 4; i++) if (n + i < p.N) dst[i] = v[i];
            }
        }
    });
}

// The outputs from the registers, where N is a multiple of 8 and rows of y are 16-byte aligned.  Of 16-bit outputs two lanes exchange a quad each, so that every lane stores 16 bytes and a slot's
// columns come in pieces of 32 or 64.  Everything that is the same for the whole launch is decided outside.  ACT: an activation of the ReLU family.
template <int FR, int WN, int WM, int FN, int FM, bool SCALED, int YT, bool GATED, bool ACT, class AccT>
__device__ __forceinline__ void lin_finish_registers(const LinearParams& p, const LinTile& tile, int n0, int g, int wn, const AccT (&acc)[FN][FM], const int (&slot)[FM], const float* wmul) {
    typedef LinQuads<FR, FN, FM> L;
    constexpr int ZN = GATED ? L::N / 2 : L::N, CW = L::CW, ES = YT == SM_F32 ? 4 : 2;   // quads of outputs
    const int first = n0 + ZN / L::Q * FR * wn;                                      // first column of this wave
    const int lane_col = YT == SM_F32 ? 4 * g : CW * (g & 1) + 8 * (g >> 1);
    const bool relu = p.act == SM_ACT_RELU;
    floatx4 add[L::N];
    if (p.bias) {
        const float* bias = p.bias + (long long)tile.e * p.w_rows;
        sm_static_for<0, ZN>([&](auto index) {
            constexpr int j = decltype(index)::value;
            const int n = first + CW * j + 4 * g, at = n < p.N ? n : p.N - 4;       // (behind the last column: not stored)
            __builtin_memcpy(&add[j], bias + at, 16);
            if constexpr (GATED) __builtin_memcpy(&add[ZN + j], bias + at + p.N, 16);
        });
    } else {
#pragma unroll
        for (int j = 0; j < L::N; j++) add[j] = floatx4{0, 0, 0, 0};
    }
    auto output = [&](auto index, int b) {                                          // quad j of the outputs
        constexpr int j = decltype(index)::value;
        if constexpr (GATED) {
            constexpr int at = j / L::UP * 2 * L::UP + j % L::UP;
            const floatx4 z = lin_quad<FR, FN, FM, SCALED, at>(acc, b, wmul) + add[j], u = lin_quad<FR, FN, FM, SCALED, at + L::UP>(acc, b, wmul) + add[ZN + j];
            return floatx4{lin_silu(z[0]) * u[0], lin_silu(z[1]) * u[1], lin_silu(z[2]) * u[2], lin_silu(z[3]) * u[3]};
        } else {
            floatx4 z = lin_quad<FR, FN, FM, SCALED, j>(acc, b, wmul) + add[j];
            if constexpr (ACT) {
#pragma unroll
                for (int i = 0; i < 4; i++) z[i] = z[i] < 0.f ? (relu ? 0.f : z[i] * p.slope) : z[i];
            }
            return z;
        }
    };
#pragma unroll
    for (int b = 0; b < FM; b++) {
        if (slot[b] >= tile.rows) continue;
        char* dst = (char*)p.y + ((tile.row0 + slot[b]) * p.y_ld + first + lane_col) * ES;
        const int left = p.N - first - lane_col;                                     // columns that exist from this lane's first on
        if constexpr (YT == SM_F32) {
            sm_static_for<0, ZN>([&](auto index) { constexpr int j = decltype(index)::value; const floatx4 v = output(index, b); if (CW * j < left) *(floatx4*)(dst + CW * j * 4) = v; });
        } else {
            sm_static_for<0, ZN / 2>([&](auto pair) {
                constexpr int j = 2 * decltype(pair)::value;
                unsigned h[2][2];
                auto round = [&](floatx4 z, unsigned* to) {
                    if constexpr (YT == SM_F16) { const half4_t t = {(half_t)z[0], (half_t)z[1], (half_t)z[2], (half_t)z[3]}; __builtin_memcpy(to, &t, 8); }
                    else { const bf16x4_t t = {(bf16_t)z[0], (bf16_t)z[1], (bf16_t)z[2], (bf16_t)z[3]}; __builtin_memcpy(to, &t, 8); }
                };
                round(output(std::integral_constant<int, j>(), b), h[0]); round(output(std::integral_constant<int, j + 1>(), b), h[1]);
                // odd lane groups give their quad j for the quad j + 1 of the group before: even ones then hold eight columns of the one, odd ones of the other
                intx4_t v;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const auto s = FR == 16 ? __builtin_amdgcn_permlane16_swap(h[0][i], h[1][i], false, false) : __builtin_amdgcn_permlane32_swap(h[0][i], h[1][i], false, false);
                    v[i] = (int)s[0]; v[2 + i] = (int)s[1];
                }
                if (CW * j < left) *(intx4_t*)(dst + CW * j * 2) = v;
            });
        }
    }
}

// Other activations, other N, other rows of y: through LDS, the fp32 tile in chunks of four columns, xor-ed with the slot; a thread takes eight consecutive columns.  BYTES of LDS, all of it free
// once every wave is here.  (8192 x 8192 outputs of K = 512 in MX4: 62 us this way, 48 from the registers, 30 without the stores.)
template <int FR, int WN, int WM, int FN, int FM, int BYTES, bool SCALED, class AccT>
__device__ __forceinline__ void lin_finish_lds(const LinearParams& p, const LinTile& tile, int n0, AccT (&acc)[FN][FM], char* lds, const float* wmul) {
    constexpr int BN = FR * FN * WN, THREADS = 64 * WN * WM;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & (FR - 1), g = lane / FR, wn = wave % WN, wm = wave / WN;
    const int cols = p.gated ? BN / 2 : BN;
    constexpr int PB = BYTES / (BN * 4) / (FR * WM) < FM ? BYTES / (BN * 4) / (FR * WM) : FM;   // slot groups of a wave that fit at once
    const float* bias = p.bias ? p.bias + (long long)tile.e * p.w_rows : nullptr;
#pragma unroll
    for (int b0 = 0; b0 < FM; b0 += PB) {
        __syncthreads();
#pragma unroll
        for (int a = 0; a < FN; a++)
#pragma unroll
            for (int q = 0; q < FR * FR / 256; q++) {
                const int j = (wn * FN + a) * (FR / 4) + 2 * q + g;                        // chunk of four columns
                floatx4 m = {1, 1, 1, 1};
                if constexpr (SCALED) m = *(const floatx4*)(wmul + 4 * j);
#pragma unroll
                for (int b = 0; b < PB; b++) {
                    const AccT v = acc[a][b0 + b];
                    *(floatx4*)(lds + ((wm * PB + b) * FR + r) * BN * 4 + ((j ^ (r & 15)) << 4)) = floatx4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]} * m;
                }
            }
        __syncthreads();
        const int per = cols / 8;
        for (int o = tid; o < PB * WM * FR * per; o += THREADS) {
            const int l = o / per, c = o - l * per, n = n0 + c * 8;                 // LDS row, group of eight columns
            const int slot = (l / (FR * PB) * FM + b0) * FR + l % (FR * PB);
            if (slot >= tile.rows || n >= p.N) continue;
            const char* row = lds + l * BN * 4;
            const int j = p.gated ? (c >> 1) * 8 + (c & 1) * 2 : 2 * c, x = l & 15;
            float v[8];
            auto get = [&](int ch, float* q, long long up) {
                const floatx4 q0 = *(const floatx4*)(row + ((ch ^ x) << 4)), q1 = *(const floatx4*)(row + (((ch + 1) ^ x) << 4));
#pragma unroll
                for (int i = 0; i < 4; i++) { q[i] = q0[i]; q[4 + i] = q1[i]; }
                if (bias) {
                    if (n + 8 <= p.N) {
                        float t[8]; __builtin_memcpy(t, bias + n + up, 32);
#pragma unroll
                        for (int i = 0; i < 8; i++) q[i] += t[i];
                    } else for (int i = 0; i < 8; i++) if (n + i < p.N) q[i] += bias[n + i + up];
                }
            };
            get(j, v, 0);
            if (p.gated) {
                float u[8]; get(j + 4, u, p.N);
                for (int i = 0; i < 8; i++) v[i] = lin_silu(v[i]) * u[i];
            } else if (p.act > SM_ACT_PRELU) {
                for (int i = 0; i < 8; i++) v[i] = sm_act_other(v[i], p.act, p.slope);
            } else if (p.act != SM_ACT_NONE) {
                const float slope = p.act == SM_ACT_RELU ? 0.f : p.slope;
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = v[i] < 0.f ? (p.act == SM_ACT_RELU ? 0.f : v[i] * slope) : v[i];
            }
            const long long out = (tile.row0 + slot) * p.y_ld + n;
            if (p.y_vec && n + 8 <= p.N) lin_store8(p.y, out, v, p.y_type);
            else for (int i = 0; i < 8; i++) if (n + i < p.N) lin_store1(p.y, out + i, v[i], p.y_type);
        }
    }
}

template <int XK, int FR, int WN, int WM, int FN, int FM, int BYTES, bool SCALED, class AccT>
__device__ __forceinline__ void lin_finish(const LinearParams& p, const LinTile& tile, int split, int n0, AccT (&acc)[FN][FM], char* lds, const float* wmul) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane & (FR - 1), g = lane / FR, wn = wave % WN, wm = wave / WN;
    if constexpr (SCALED) __syncthreads();                                          // (wmul, of a product without a step)
    int slot[FM]; bool dead[FM], any = false;
#pragma unroll
    for (int b = 0; b < FM; b++) {
        slot[b] = FR * (wm * FM + b) + r;
        dead[b] = p.rows && lin_slot_row(p, tile, slot[b]) < 0;
        any |= dead[b];
    }
    if (__any(any)) {                                                               // slots without a row of x: zero, also under weights that are infinite or NaN
#pragma unroll
        for (int a = 0; a < FN; a++)
#pragma unroll
            for (int b = 0; b < FM; b++)
#pragma unroll
                for (int i = 0; i < FR * FR / 64; i++) acc[a][b][i] = dead[b] ? 0.f : acc[a][b][i];
    }
    const int row0 = FR * wn * FN + 4 * g;
    if constexpr (FR == 32 && FM == 1) if (p.splits > 1) { lin_finish_split<FR, FN, FM, SCALED>(p, tile, split, n0, row0, acc, slot, wmul + row0); return; }
    if (p.y_vec && p.N % 8 == 0 && p.act <= SM_ACT_PRELU) {
        if (wm * FM * FR >= tile.rows) return;
        auto go = [&](auto type) {
            constexpr int YT = decltype(type)::value;
            if (p.gated) lin_finish_registers<FR, WN, WM, FN, FM, SCALED, YT, true, false>(p, tile, n0, g, wn, acc, slot, wmul + row0);
            else if (p.act != SM_ACT_NONE) lin_finish_registers<FR, WN, WM, FN, FM, SCALED, YT, false, true>(p, tile, n0, g, wn, acc, slot, wmul + row0);
            else lin_finish_registers<FR, WN, WM, FN, FM, SCALED, YT, false, false>(p, tile, n0, g, wn, acc, slot, wmul + row0);
        };
        if (p.y_type == SM_F32) go(std::integral_constant<int, SM_F32>());
        else if (p.y_type == SM_F16) go(std::integral_constant<int, SM_F16>());
        else if constexpr (XK != SM_F16) go(std::integral_constant<int, SM_BF16>());
        return;
    }
    lin_finish_lds<FR, WN, WM, FN, FM, BYTES, SCALED>(p, tile, n0, acc, lds, wmul);
}

// the eight 16-bit elements of v without the first n, zeros behind them
__device__ __forceinline__ intx4_t lin_drop(intx4_t v, int n) {
    typedef unsigned long long ull;
    const ull lo = (unsigned)v[0] | (ull)(unsigned)v[1] << 32, hi = (unsigned)v[2] | (ull)(unsigned)v[3] << 32;
    const int s = 16 * n, t = s & 63;
    const ull a = t ? (lo >> t) | (hi << (64 - t)) : lo, b = hi >> t;
    const ull l = s < 64 ? a : s < 128 ? b : 0, h = s < 64 ? b : 0;
    return intx4_t{(int)l, (int)(l >> 32), (int)h, (int)(h >> 32)};
}

template <int XK, int WK, int FR, int WN, int WM, int FN, int FM, bool DMA> struct LinTileShape {
    static constexpr int THREADS = 64 * WN * WM, BN = FR * FN * WN, BM = FR * FM * WM;
    static constexpr bool DEQ = WK == SM_MX4 && XK != SM_MX4, MX = XK == SM_MX4;
    static constexpr int STAGE = (BN + BM) * 128;
    static constexpr int SCALES = MX ? 2 * (BN + BM) * 8 : DEQ ? BN * 4 : 0;
    static constexpr int LDS = 2 * STAGE + SCALES;
};

template <int XK, int WK, int FR, int WN, int WM, int FN, int FM, bool DMA>
__global__ __launch_bounds__(64 * WN * WM) void lin_tile_kernel(LinearParams p) {
    typedef LinTileShape<XK, WK, FR, WN, WM, FN, FM, DMA> S;
    constexpr int THREADS = S::THREADS, BN = S::BN, BM = S::BM, WAVES = WN * WM;
    constexpr bool DEQ = S::DEQ, MX = S::MX;
    __shared__ __align__(16) char lds[S::LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & (FR - 1), g = lane / FR;

    int split, nt;
    constexpr bool HALVES = FR == 16 && DMA && !DEQ && !MX;                         // (the others' waves have work for each other: a half takes as long)
    const LinTile tile = lin_pick_tile<HALVES>(p, BM, &split, &nt);
    if (tile.rows == 0) return;
    const int row_bytes = MX || DEQ ? 16 * ((p.K + 31) >> 5) : 2 * p.K;             // of a weight row
    const int x_bytes = MX ? row_bytes : 2 * p.K;
    const int every = (x_bytes + 127) >> 7, nb = (p.K + 31) >> 5;
    const int first = (int)((long long)every * split / p.splits), steps = (int)((long long)every * (split + 1) / p.splits);   // the steps first .. steps - 1 of all
    const int cols = p.gated ? BN / 2 : BN, n0 = nt * cols;

    auto weight_row = [&](int j) { return lin_weight_row(p, n0, j); };
    auto slot_row = [&](int j) { return lin_slot_row(p, tile, j); };
    const char* wexp = p.w + tile.e * p.w_es;

    // ---- LDS-DMA: instruction q of a wave fills rows 8 q .. 8 q + 7 of a stage
    constexpr int QW = DEQ ? 0 : BN / 8 / WAVES, QX = BM / 8 / WAVES;
    unsigned woff[QW > 0 ? QW : 1], xoff[QX];                                        // bytes from the expert's weights / the tile's rows: lin_tile_fits() holds them below 2^32
    const char* xbase = p.rows ? p.x : p.x + tile.row0 * p.x_ld;
    const int chunk = (lane & 7) ^ (lane >> 3);
    auto swz = [](int row) { return FR == 32 ? row >> 4 & 1 : 0; };
    if constexpr (!DEQ) {
#pragma unroll
        for (int i = 0; i < QW; i++) woff[i] = (unsigned)(weight_row((wave * QW + i) * 8 + (lane >> 3)) * p.w_ld);
    }
#pragma unroll
    for (int i = 0; i < QX; i++) { const long long s = slot_row((wave * QX + i) * 8 + (lane >> 3)); xoff[i] = (unsigned)((s < 0 ? 0 : p.rows ? s : s - tile.row0) * p.x_ld); }
    const unsigned lds0 = lin_lds_addr(lds);
    constexpr int QT = QW + QX;
    auto fill = [&](int t, int i) {                                                 // instruction i of QT
        const int q = i < QW ? wave * QW + i : wave * QX + i - QW;
        int k = t * 128 + (chunk ^ swz(q * 8)) * 16; if (k > x_bytes - 16) k = x_bytes - 16;   // behind the end: the row's last chunk again (masked when it is read)
        const unsigned st = lds0 + (t & 1) * S::STAGE;
        if (i < QW) lin_dma16(wexp, woff[i < QW ? i : 0] + k, st + (wave * QW + i) * 1024);
        else lin_dma16(xbase, xoff[i - QW] + k, st + BN * 128 + (wave * QX + i - QW) * 1024);
    };

    // ---- what goes through registers: loaded two steps before it is read, stored one step before
    intx4_t wreg[DMA || QW == 0 ? 1 : QW], xreg[DMA ? 1 : QX];                      // rows that are not 16-byte aligned (odd K, a slice of a wider tensor)
    constexpr int DB = DEQ ? BN * 2 / THREADS : 1;                                  // MX4 weights under a 16-bit x: a thread turns blocks of 32 into 64 bytes of its row
    intx4_t code[DB]; int sbyte[DB], stop[DB];
    const char* csrc[DB]; const unsigned char* ssrc[DB];
    float* wmul = (float*)(lds + 2 * S::STAGE);
    if constexpr (DEQ) {
#pragma unroll
        for (int i = 0; i < DB; i++) {
            const int j = i * (THREADS / 2) + (tid >> 1);
            const long long row = weight_row(j);
            csrc[i] = wexp + row * p.w_ld; ssrc[i] = p.ws + tile.e * p.ws_es + row * p.ws_ld;
            stop[i] = 127;
            if constexpr (XK == SM_F16) {                                           // relative to the row's largest scale; a row that reaches too far is marked by a negative factor
                LinSpread all;
                for (int b = 16 * (tid & 1); b < nb && nb >= 16; b += 32) {
                    intx4_t v; __builtin_memcpy(&v, ssrc[i] + (b < nb - 16 ? b : nb - 16), 16);
                    all.look(v[0]); all.look(v[1]); all.look(v[2]); all.look(v[3]);
                }
                for (int b = 0; b < nb && nb < 16; b++) all.look(ssrc[i][b] * 0x01010101u);
                int top = all.top(); const int low = all.low();
                const int o = __shfl_xor(top, 1); top = top > o ? top : o;
                if (top == 255) { top = 0; for (int b = 0; b < nb; b++) top = lin_top_of(top, ssrc[i][b]); }   // a NaN block: the largest of the others
                if (top < 14) top = 14;
                int far = 0;
                if (top - low > LIN_REACH)
                    for (int b = 0; b < nb; b++)
                        if (lin_relative(ssrc[i][b], top) < 140 - LIN_REACH) { intx4_t c; __builtin_memcpy(&c, csrc[i] + 16ll * b, 16); far |= (c[0] | c[1] | c[2] | c[3]) & 0x77777777; }
                far |= __shfl_xor(far, 1);                                          // (each of the two threads has seen half of the scales)
                stop[i] = top;
                if (!(tid & 1)) wmul[j] = far ? -1.f : lin_top_scale(top);
            }
        }
    }
    // scales of MX4 operands: the eight bytes of a step of each row
    constexpr int SB = MX ? (BN + BM + THREADS - 1) / THREADS : 1;
    unsigned long long sreg[SB]; const unsigned char* srow[SB];
    if constexpr (MX) {
#pragma unroll
        for (int i = 0; i < SB; i++) {
            const int j = i * THREADS + tid < BN + BM ? i * THREADS + tid : BN + BM - 1;   // (threads to spare repeat the last row)
            if (j < BN) srow[i] = p.ws + tile.e * p.ws_es + weight_row(j) * p.ws_ld;
            else { const long long s = slot_row(j - BN); srow[i] = p.xs + (s < 0 ? 0 : s) * p.xs_ld; }
        }
    }
    auto load_staged = [&](int t, auto loop) {                                      // in the loop without a branch: the compiler would move products across it, out of their phase
        if constexpr (MX) {
            const int at = 8 * t < nb - 8 ? 8 * t : nb - 8;                         // the last ones of a row as its last eight bytes
            if (decltype(loop)::value || nb >= 8) {
#pragma unroll
                for (int i = 0; i < SB; i++) __builtin_memcpy(&sreg[i], srow[i] + at, 8);
            } else {                                                                // (a row of one step)
#pragma unroll
                for (int i = 0; i < SB; i++) {
                    sreg[i] = 0;
#pragma unroll
                    for (int b = 0; b < 7; b++) if (b < nb) sreg[i] |= (unsigned long long)srow[i][b] << (8 * b);
                }
            }
        }
        if constexpr (DEQ) {
#pragma unroll
            for (int i = 0; i < DB; i++) {
                const int b = 2 * t + (tid & 1), at = b < nb ? b : nb - 1;
                code[i] = *(const intx4_t*)(csrc[i] + 16ll * at); sbyte[i] = b < nb ? ssrc[i][at] : 0;   // (behind the end: finite, under zeros of x)
            }
        }
        if constexpr (!DMA) {
            auto at = [&](int q) { const int k = t * 64 + (chunk ^ swz(q * 8)) * 8; return 2ll * (k < p.K - 8 ? k : p.K - 8); };   // the last ones of a row as its last eight elements
            if constexpr (!DEQ) {
#pragma unroll
                for (int i = 0; i < QW; i++) __builtin_memcpy(&wreg[i], wexp + woff[i] + at(wave * QW + i), 16);
            }
#pragma unroll
            for (int i = 0; i < QX; i++) __builtin_memcpy(&xreg[i], xbase + xoff[i] + at(wave * QX + i), 16);
        }
    };
    auto store_staged = [&](int t, auto end) {                                      // end: t may be the last step of a row
        if constexpr (MX) {
            const int over = nb >= 8 && 8 * t > nb - 8 ? 8 * t - (nb - 8) : 0;      // bytes of the step before, shifted out; behind the end (codes 0) scale 0
#pragma unroll
            for (int i = 0; i < SB; i++) {
                const unsigned long long v = sreg[i] >> (8 * over);
                const unsigned lo = (unsigned)v, hi = (unsigned)(v >> 32);
                // the bytes of a lane group side by side (one LDS read a step): blocks g, 4 + g of fragments of 16 rows, g, 2 + g, 4 + g, 6 + g of 32
                const unsigned a = FR == 16 ? __builtin_amdgcn_perm(hi, lo, 0x05010400) : __builtin_amdgcn_perm(hi, lo, 0x06040200);
                const unsigned b = FR == 16 ? __builtin_amdgcn_perm(hi, lo, 0x07030602) : __builtin_amdgcn_perm(hi, lo, 0x07050301);
                *(unsigned long long*)(lds + 2 * S::STAGE + ((t & 1) * (BN + BM) + (i * THREADS + tid < BN + BM ? i * THREADS + tid : BN + BM - 1)) * 8) = a | (unsigned long long)b << 32;
            }
        }
        if constexpr (DEQ) {
            char* st = lds + (t & 1) * S::STAGE;
#pragma unroll
            for (int i = 0; i < DB; i++) {
                const int j = i * (THREADS / 2) + (tid >> 1);
                int byte = sbyte[i];
                if constexpr (XK == SM_F16) byte = lin_relative(byte, stop[i]);
                const float s = mx4_scale(byte);
#pragma unroll
                for (int q = 0; q < 4; q++) *(intx4_t*)(st + j * 128 + ((((tid & 1) * 4 + q) ^ (j & 7) ^ swz(j)) << 4)) = mx4_to16<XK>(code[i][q], s);
            }
        }
        if constexpr (!DMA) {
            char* st = lds + (t & 1) * S::STAGE + lane * 16;
            auto over = [&](int q) { const int k = t * 64 + (chunk ^ swz(q * 8)) * 8; return k > p.K - 8 ? k - (p.K - 8) : 0; };   // elements before k in the eight; behind the row's end zeros
            if constexpr (!DEQ) {
#pragma unroll
                for (int i = 0; i < QW; i++) { if constexpr (decltype(end)::value) wreg[i] = lin_drop(wreg[i], over(wave * QW + i)); *(intx4_t*)(st + (wave * QW + i) * 1024) = wreg[i]; }
            }
#pragma unroll
            for (int i = 0; i < QX; i++) { if constexpr (decltype(end)::value) xreg[i] = lin_drop(xreg[i], over(wave * QX + i)); *(intx4_t*)(st + BN * 128 + (wave * QX + i) * 1024) = xreg[i]; }
        }
    };
    // ---- the products of a step in four phases (fragments of 32 rows: one for each 32 bytes of K; of 16 rows: one for each 64 bytes of K and each half of the wave's weight rows; 128-row tiles of
    // them: two phases); a phase's fragments are read during the phase before it (over the step boundary too)
    typedef float AccT __attribute__((ext_vector_type(FR * FR / 64)));
    constexpr int GA = FR == 32 ? FN : 4, HA = FN / GA, PH = (FR == 32 ? 4 : 2) * HA;
    const int wn = wave % WN, wm = wave / WN;                                       // this wave's part of the tile
    AccT acc[FN][FM];
#pragma unroll
    for (int a = 0; a < FN; a++)
#pragma unroll
        for (int b = 0; b < FM; b++)
#pragma unroll
            for (int i = 0; i < FR * FR / 64; i++) acc[a][b][i] = 0.f;
    intx4_t wf[2][GA], xf[2][FM];
    int wall[MX ? FN : 1], xall[MX ? FM : 1], wsc[2][MX && HA == 1 ? GA : 1], xsc[2][MX ? FM : 1];   // scale bytes: of a lane's blocks of the step, and of the phase
    auto read = [&](int t, auto phase, bool masked) {
        constexpr int P = decltype(phase)::value, H = P / HA, A = P % HA, WB = P & 1, XB = H & 1;
        const int ch = H * (64 / FR) + g;                                           // this lane's chunk of the row
        const char* st = lds + (t & 1) * S::STAGE + r * 128 + ((ch ^ (lane & 7) ^ swz(r)) << 4);
#pragma unroll
        for (int a = 0; a < GA; a++) wf[WB][a] = *(const intx4_t*)(st + (wn * FN + A * GA + a) * (FR * 128));
        if constexpr (A == 0) {
#pragma unroll
            for (int b = 0; b < FM; b++) xf[XB][b] = *(const intx4_t*)(st + (BN / FR + wm * FM + b) * (FR * 128));
        }
        if constexpr (MX) {
            typedef std::conditional_t<FR == 16, unsigned short, int> Word;
            const char* sc = lds + 2 * S::STAGE + (t & 1) * (BN + BM) * 8 + r * 8 + g * (FR / 8);
            if constexpr (H == 0) {
#pragma unroll
                for (int a = 0; a < GA; a++) wall[A * GA + a] = *(const Word*)(sc + (wn * FN + A * GA + a) * (FR * 8));
                if constexpr (A == 0) {
#pragma unroll
                    for (int b = 0; b < FM; b++) xall[b] = *(const Word*)(sc + (BN / FR + wm * FM + b) * (FR * 8));
                }
            }
            if constexpr (HA == 1) {                                                // (copies: the next step's are read while the last phase runs)
#pragma unroll
                for (int a = 0; a < GA; a++) wsc[WB][a] = wall[a] >> (8 * H);
            }
            if constexpr (A == 0) {
#pragma unroll
                for (int b = 0; b < FM; b++) xsc[XB][b] = xall[b] >> (8 * H);
            }
        }
        if (masked) {                                                               // chunks behind the end of the row
            const bool dead = t * 128 + ch * 16 >= x_bytes;
#pragma unroll
            for (int a = 0; a < GA; a++) wf[WB][a] = dead ? intx4_t{0, 0, 0, 0} : wf[WB][a];
            if constexpr (A == 0) {
#pragma unroll
                for (int b = 0; b < FM; b++) xf[XB][b] = dead ? intx4_t{0, 0, 0, 0} : xf[XB][b];
            }
        }
    };
    auto products = [&](auto phase, auto between) {                                 // between(a): behind the a-th row of tiles
        constexpr int P = decltype(phase)::value, A = P % HA, WB = P & 1, XB = (P / HA) & 1;
        sm_static_for<0, GA>([&](auto ai) {
            constexpr int a = decltype(ai)::value;
            if constexpr (a == 1) __builtin_amdgcn_s_setprio(1);                    // the wave that has its fragments goes first, the other one of the SIMD reads: 1 - 2 %
#pragma unroll
            for (int b = 0; b < FM; b++) {
                AccT& c = acc[A * GA + a][b];
                if constexpr (MX && HA == 1) c = lin_mma4<0>(wf[WB][a], wsc[WB][a], xf[XB][b], xsc[XB][b], c);
                else if constexpr (MX) c = lin_mma4<P / HA>(wf[WB][a], wall[A * GA + a], xf[XB][b], xsc[XB][b], c);
                else c = lin_mma16<XK>(wf[WB][a], xf[XB][b], c);
            }
            between(a);
            if constexpr (a == GA - 1) __builtin_amdgcn_s_setprio(0);
        });
    };
    typedef std::integral_constant<int, 0> First; typedef std::integral_constant<int, PH - 1> Last;
    const bool ragged = DMA && (x_bytes & 127) && steps == every;
    int t = first;
    if (steps > first) {
        if constexpr (DMA) {
#pragma unroll
            for (int i = 0; i < QT; i++) fill(first, i);
        }
        load_staged(first, std::false_type()); store_staged(first, std::true_type());
        if (steps > first + 1) {
            if constexpr (DMA) {
#pragma unroll
                for (int i = 0; i < QT / 2; i++) fill(first + 1, i);
            }
            load_staged(first + 1, std::false_type()); store_staged(first + 1, std::true_type());
        }
        if (steps > first + 2) load_staged(first + 2, std::false_type());
        lin_arrive();
        if constexpr (DEQ && XK == SM_F16) {
            float least = 0.f;
#pragma unroll
            for (int j = 0; j < BN; j += 64) { const float m = wmul[j + lane]; least = m < least ? m : least; }
            if (__any(least < 0.f)) {                                               // (every wave sees the same)
                lin_arrive();
                if (tid < BN) wmul[tid] = 1.f;
                const char* xr[FM]; int xk[FM];
#pragma unroll
                for (int b = 0; b < FM; b++) { const long long row = slot_row(FR * (wm * FM + b) + r); xr[b] = p.x + (row < 0 ? 0 : row) * p.x_ld; xk[b] = row < 0 ? 0 : p.K; }
#pragma unroll
                for (int a = 0; a < FN; a++) {
                    const long long row = weight_row(FR * (wn * FN + a) + r);
                    lin_exact_blocks<FR, FM>(wexp + row * p.w_ld, p.ws + tile.e * p.ws_es + row * p.ws_ld, xr, xk, 2 * first, 2 * steps < nb ? 2 * steps : nb,
                                             [&](int b, intx4_t w, intx4_t x) { acc[a][b] = lin_mma16<SM_BF16>(w, x, acc[a][b]); },
                                             [&] {
#pragma unroll
                                                 for (int b = 0; b < FM; b++) acc[a][b] = acc[a][b] * 0x1p64f * 0x1p64f;
                                             });
                }
                t = steps;
            }
        }
        if (t < steps) read(first, First(), ragged && steps == first + 1);
    }
    auto step = [&](int t, auto has1, auto has2, auto end2) {                       // has1, has2: steps t + 1, t + 2 exist; end2: t + 2 may be the last
        constexpr bool MORE = decltype(has1)::value, MORE2 = decltype(has2)::value;
        sm_static_for<0, PH - 1>([&](auto phase) {
            constexpr int P = decltype(phase)::value;
            products(phase, [&](int a) {
                if (a == 0) { __builtin_amdgcn_sched_barrier(0); read(t, std::integral_constant<int, P + 1>(), !MORE && ragged); __builtin_amdgcn_sched_barrier(0); }
                if constexpr (DMA && P == 0 && MORE) {                              // the second half of the next step's fill, one instruction at a time
#pragma unroll
                    for (int i = QT / 2 + a * (QT - QT / 2) / GA; i < QT / 2 + (a + 1) * (QT - QT / 2) / GA; i++) fill(t + 1, i);
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (MORE) {
            lin_arrive();                                                           // step t + 1 is in LDS for everybody; everybody has read the whole of step t
            if constexpr (MORE2) { store_staged(t + 2, end2); load_staged(t + 3 < steps ? t + 3 : steps - 1, std::true_type()); }
        }
        products(Last(), [&](int a) {
            if constexpr (MORE) if (a == 0) { __builtin_amdgcn_sched_barrier(0); read(t + 1, First(), !MORE2 && ragged); __builtin_amdgcn_sched_barrier(0); }
            if constexpr (DMA && MORE2) {                                           // the first half of the fill behind it
#pragma unroll
                for (int i = a * (QT / 2) / GA; i < (a + 1) * (QT / 2) / GA; i++) fill(t + 2, i);
            }
        });
        __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (DMA && !DEQ && !MX) {
        // a wave whose slots lie behind the tile's last one (the end of a group) only fills; the four SIMDs hold waves of all parts, so that the others run faster
        if (wm * FM * FR >= tile.rows) {
            for (; t + 1 < steps; t++) {
#pragma unroll
                for (int i = QT / 2; i < QT; i++) fill(t + 1, i);
                lin_arrive();
                if (t + 2 < steps) {
#pragma unroll
                    for (int i = 0; i < QT / 2; i++) fill(t + 2, i);
                }
            }
            t = steps;
        }
    }
#pragma unroll 1
    for (; t + (DMA ? 2 : 3) < steps; t++) step(t, std::true_type(), std::true_type(), std::false_type());
    if constexpr (!DMA) if (t + 2 < steps) { step(t, std::true_type(), std::true_type(), std::true_type()); t++; }
    if (t + 1 < steps) { step(t, std::true_type(), std::false_type(), std::false_type()); t++; }
    if (t < steps) step(t, std::false_type(), std::false_type(), std::false_type());

    lin_finish<XK, FR, WN, WM, FN, FM, 2 * S::STAGE, DEQ && XK == SM_F16>(p, tile, split, n0, acc, lds, wmul);
}

template <int XK, int WK, int FR, int WN, int WM, int FN, int FM, bool DMA> static int lin_tile(const LinearParams& q, hipStream_t s) {
    typedef LinTileShape<XK, WK, FR, WN, WM, FN, FM, DMA> S;
    LinearParams p = q;
    const int cols = p.gated ? S::BN / 2 : S::BN;
    p.n_tiles = (p.N + cols - 1) / cols;
    p.m_tiles = lin_row_tiles(p, S::BM);
    const long long blocks = (p.m_tiles * p.n_tiles + 7) / 8 * 8 * p.splits + (FR == 16 ? SM_NUM_CU / 2 : 0);   // (and the second halves of lin_pick_tile)
    SM_REQUIRE(lin_one_launch(blocks, S::THREADS), "linear: %lld row tiles x %d column tiles exceed one launch", p.m_tiles, p.n_tiles);
    lin_tile_kernel<XK, WK, FR, WN, WM, FN, FM, DMA><<<dim3((unsigned)blocks), S::THREADS, 0, s>>>(p);
    SM_LAUNCH_CHECK();
    return SM_OK;
}
