// smelter_amd/csrc/kernels/linear_tile.hpp — linear layers on MANY rows: tiles of BN weight rows x BM slots through LDS, 128 bytes of K at a time.
//
// Both operands lie in LDS as rows of 128 bytes (64 16-bit elements, or 8 MX4 blocks = 256 elements), filled by the LDS-DMA without passing a register; 16-byte chunk c of row r sits at place
// c ^ (r & 7), so that the 16 rows a fragment read touches spread over all banks.  The weights are the first operand of the matrix instruction: a lane then holds four consecutive columns of one
// slot, which it stores together.  A 32 x 32 x 16 product of 16-bit fragments and a 32 x 32 x 64 product of MX4 fragments read the same bytes and take the same cycles, so both kinds share the
// kernel; the MX4 one adds the scale bytes.  MX4 weights under a 16-bit x become 16-bit values on their way into LDS.
#pragma once
#include "linear.hpp"

// 16 bytes per lane from base + off -> lds + 16 * lane (base and lds wave-uniform); completion: s_waitcnt vmcnt
__device__ __forceinline__ void lin_dma16(const char* base, unsigned off, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(off), "s"(base), "s"(lds));
}
__device__ __forceinline__ unsigned lin_lds_addr(const void* p) { return (unsigned)(size_t)(const __attribute__((address_space(3))) void*)p; }
__device__ __forceinline__ void lin_arrive() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int XK, int WK, int WN, int WM, int FN, int FM, bool DMA> struct LinTileShape {
    static constexpr int THREADS = 64 * WN * WM, BN = 32 * FN * WN, BM = 32 * FM * WM;
    static constexpr bool DEQ = WK == SM_MX4 && XK != SM_MX4, MX = XK == SM_MX4;
    static constexpr int STAGE = (BN + BM) * 128;
    static constexpr int SCALES = MX ? 2 * (BN + BM) * 8 : DEQ ? BN * 4 : 0;
    static constexpr int LDS = 2 * STAGE + SCALES;
};

template <int XK, int WK, int WN, int WM, int FN, int FM, bool DMA>
__global__ __launch_bounds__(64 * WN * WM) void lin_tile_kernel(LinearParams p) {
    typedef LinTileShape<XK, WK, WN, WM, FN, FM, DMA> S;
    constexpr int THREADS = S::THREADS, BN = S::BN, BM = S::BM, WAVES = WN * WM;
    constexpr bool DEQ = S::DEQ, MX = S::MX;
    __shared__ __align__(16) char lds[S::LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5;

    // ---- which tile: consecutive tiles stay on one XCD (blocks are dealt to the 8 XCDs in turn), in squares of up to 8 row tiles, so that an XCD's L2 holds what its CUs read together
    const LinTile all = lin_find_tile(p, BM, 0, true);
    const long long total = all.total * p.n_tiles;
    long long id;
    {
        const long long b = blockIdx.x; const int xcd = (int)(b & 7); const long long q = total >> 3; const int rem = (int)(total & 7);
        if ((b >> 3) >= q + (xcd < rem ? 1 : 0)) return;
        id = xcd * q + (xcd < rem ? xcd : rem) + (b >> 3);
    }
    const long long band = id / (8ll * p.n_tiles);
    const int in = (int)(id - band * 8 * p.n_tiles), high = (int)(all.total - band * 8 < 8 ? all.total - band * 8 : 8);
    const int nt = in / high;
    const LinTile tile = lin_find_tile(p, BM, band * 8 + in - nt * high, false);
    if (tile.rows == 0) return;
    const int row_bytes = MX || DEQ ? 16 * ((p.K + 31) >> 5) : 2 * p.K;             // of a weight row
    const int x_bytes = MX ? row_bytes : 2 * p.K;
    const int steps = (x_bytes + 127) >> 7, nb = (p.K + 31) >> 5;
    const int cols = p.gated ? BN / 2 : BN, n0 = nt * cols;

    // weight row of tile row j: gated tiles alternate 16 gate rows and their 16 up rows
    auto weight_row = [&](int j) -> long long {
        int n = p.gated ? n0 + ((j >> 5) << 4) + (j & 15) : n0 + j;
        if (n >= p.N) n = p.N - 1;
        return n + (p.gated && (j & 16) ? (long long)p.N : 0);
    };
    auto slot_row = [&](int j) -> long long {                                       // row of x of tile slot j, -1: outside x
        long long s = tile.row0 + (j < tile.rows ? j : tile.rows - 1);
        if (p.rows) { s = p.rows[s]; if (s < 0 || s >= p.T) s = -1; }
        return s;
    };
    const char* wexp = p.w + tile.e * p.w_es;

    // ---- LDS-DMA: instruction q of a wave fills rows 8 q .. 8 q + 7 of a stage
    constexpr int QW = DEQ ? 0 : BN / 8 / WAVES, QX = BM / 8 / WAVES;
    unsigned woff[QW > 0 ? QW : 1], xoff[QX];                                        // bytes from the expert's weights / the tile's rows: lin_tile_fits() holds them below 2^32
    const char* xbase = p.rows ? p.x : p.x + tile.row0 * p.x_ld;
    const int chunk = (lane & 7) ^ (lane >> 3);
    if constexpr (!DEQ) {
#pragma unroll
        for (int i = 0; i < QW; i++) woff[i] = (unsigned)(weight_row((wave * QW + i) * 8 + (lane >> 3)) * p.w_ld);
    }
#pragma unroll
    for (int i = 0; i < QX; i++) { const long long s = slot_row((wave * QX + i) * 8 + (lane >> 3)); xoff[i] = (unsigned)((s < 0 ? 0 : p.rows ? s : s - tile.row0) * p.x_ld); }
    const unsigned lds0 = lin_lds_addr(lds);
    constexpr int QT = QW + QX;
    auto fill = [&](int t, int i) {                                                 // instruction i of QT
        int k = t * 128 + chunk * 16; if (k > x_bytes - 16) k = x_bytes - 16;       // behind the end: the row's last chunk again (masked when it is read)
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
            if constexpr (XK == SM_F16) {                                           // values relative to the row's largest scale: inside fp16's range whatever the scales are
                int top = 1;
                for (int b = tid & 1; b < nb; b += 2) { const int s = ssrc[i][b]; top = top > s ? top : s; }
                const int o = __shfl_xor(top, 1); top = top > o ? top : o;
                stop[i] = top;
                if (!(tid & 1)) wmul[j] = mx4_scale(top);
            }
        }
    }
    // scales of MX4 operands: the eight bytes of a step of each row
    constexpr int SB = MX ? (BN + BM) / THREADS : 1;
    unsigned long long sreg[SB]; const unsigned char* srow[SB];
    if constexpr (MX) {
#pragma unroll
        for (int i = 0; i < SB; i++) {
            const int j = i * THREADS + tid;
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
                code[i] = *(const intx4_t*)(csrc[i] + 16ll * at); sbyte[i] = ssrc[i][at];
            }
        }
        if constexpr (!DMA) {
            const int k = t * 64 + chunk * 8;
            if constexpr (!DEQ) {
#pragma unroll
                for (int i = 0; i < QW; i++) wreg[i] = lin_load8(wexp + woff[i], k, p.K);
            }
#pragma unroll
            for (int i = 0; i < QX; i++) xreg[i] = lin_load8(xbase + xoff[i], k, p.K);
        }
    };
    auto store_staged = [&](int t) {
        if constexpr (MX) {
            const int over = nb >= 8 && 8 * t > nb - 8 ? 8 * t - (nb - 8) : 0;      // bytes of the step before, shifted out; behind the end (codes 0) scale 0
#pragma unroll
            for (int i = 0; i < SB; i++) *(unsigned long long*)(lds + 2 * S::STAGE + ((t & 1) * (BN + BM) + i * THREADS + tid) * 8) = sreg[i] >> (8 * over);
        }
        if constexpr (DEQ) {
            char* st = lds + (t & 1) * S::STAGE;
#pragma unroll
            for (int i = 0; i < DB; i++) {
                const int j = i * (THREADS / 2) + (tid >> 1);
                int byte = sbyte[i];
                if constexpr (XK == SM_F16) { const int d = byte - stop[i] + 127; byte = byte == 255 ? 255 : d > 0 ? d : 0; }
                const float s = mx4_scale(byte);
#pragma unroll
                for (int q = 0; q < 4; q++) *(intx4_t*)(st + j * 128 + ((((tid & 1) * 4 + q) ^ (j & 7)) << 4)) = mx4_to16<XK>(code[i][q], s);
            }
        }
        if constexpr (!DMA) {
            char* st = lds + (t & 1) * S::STAGE + lane * 16;
            if constexpr (!DEQ) {
#pragma unroll
                for (int i = 0; i < QW; i++) *(intx4_t*)(st + (wave * QW + i) * 1024) = wreg[i];
            }
#pragma unroll
            for (int i = 0; i < QX; i++) *(intx4_t*)(st + BN * 128 + (wave * QX + i) * 1024) = xreg[i];
        }
    };
    // ---- the products of a step in four phases, one for each 32 bytes of K; a phase's fragments are read during the phase before it (over the step boundary too)
    constexpr int PH = 4;
    const int wn = wave / WM, wm = wave - wn * WM;                                  // this wave's part of the tile
    floatx16 acc[FN][FM];
#pragma unroll
    for (int a = 0; a < FN; a++)
#pragma unroll
        for (int b = 0; b < FM; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[a][b][i] = 0.f;
    intx4_t wf[2][FN], xf[2][FM]; int wsc[2][MX ? FN : 1], xsc[2][MX ? FM : 1];
    auto read = [&](int t, auto phase, bool masked) {
        constexpr int P = decltype(phase)::value, B = P & 1;
        const char* st = lds + (t & 1) * S::STAGE + r * 128 + (((2 * P + g) ^ (lane & 7)) << 4);
#pragma unroll
        for (int a = 0; a < FN; a++) wf[B][a] = *(const intx4_t*)(st + (wn * FN + a) * 4096);
#pragma unroll
        for (int b = 0; b < FM; b++) xf[B][b] = *(const intx4_t*)(st + (BN / 32 + wm * FM + b) * 4096);
        if constexpr (MX) {
            const unsigned char* sc = (const unsigned char*)lds + 2 * S::STAGE + (t & 1) * (BN + BM) * 8 + r * 8 + g + 2 * P;
#pragma unroll
            for (int a = 0; a < FN; a++) wsc[B][a] = sc[(wn * FN + a) * 256];
#pragma unroll
            for (int b = 0; b < FM; b++) xsc[B][b] = sc[(BN / 32 + wm * FM + b) * 256];
        }
        if (masked) {                                                               // chunks behind the end of the row
            const bool dead = t * 128 + (2 * P + g) * 16 >= x_bytes;
#pragma unroll
            for (int a = 0; a < FN; a++) wf[B][a] = dead ? intx4_t{0, 0, 0, 0} : wf[B][a];
#pragma unroll
            for (int b = 0; b < FM; b++) xf[B][b] = dead ? intx4_t{0, 0, 0, 0} : xf[B][b];
        }
    };
    auto products = [&](auto phase, auto between) {                                 // between(a): behind the a-th row of tiles
        constexpr int B = decltype(phase)::value & 1;
        sm_static_for<0, FN>([&](auto ai) {
            constexpr int a = decltype(ai)::value;
#pragma unroll
            for (int b = 0; b < FM; b++) {
                if constexpr (MX) acc[a][b] = lin_mma4(wf[B][a], wsc[B][a], xf[B][b], xsc[B][b], acc[a][b]);
                else acc[a][b] = lin_mma16<XK>(wf[B][a], xf[B][b], acc[a][b]);
            }
            between(a);
        });
    };
    typedef std::integral_constant<int, 0> First; typedef std::integral_constant<int, PH - 1> Last;
    const bool ragged = DMA && (x_bytes & 127);
    if (steps > 0) {
        if constexpr (DMA) {
#pragma unroll
            for (int i = 0; i < QT; i++) fill(0, i);
        }
        load_staged(0, std::false_type()); store_staged(0);
        if (steps > 1) {
            if constexpr (DMA) {
#pragma unroll
                for (int i = 0; i < QT / 2; i++) fill(1, i);
            }
            load_staged(1, std::false_type()); store_staged(1);
        }
        if (steps > 2) load_staged(2, std::false_type());
        lin_arrive();
        read(0, First(), ragged && steps == 1);
    }
    auto step = [&](int t, auto has1, auto has2) {                                  // has1, has2: steps t + 1, t + 2 exist
        constexpr bool MORE = decltype(has1)::value, MORE2 = decltype(has2)::value;
        sm_static_for<0, PH - 1>([&](auto phase) {
            constexpr int P = decltype(phase)::value;
            products(phase, [&](int a) {
                if (a == 0) { __builtin_amdgcn_sched_barrier(0); read(t, std::integral_constant<int, P + 1>(), !MORE && ragged); __builtin_amdgcn_sched_barrier(0); }
                if constexpr (DMA && P == 0 && MORE) {                              // the second half of the next step's fill, one instruction at a time
#pragma unroll
                    for (int i = QT / 2 + a * (QT - QT / 2) / FN; i < QT / 2 + (a + 1) * (QT - QT / 2) / FN; i++) fill(t + 1, i);
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (MORE) {
            lin_arrive();                                                           // step t + 1 is in LDS for everybody; everybody has read the whole of step t
            if constexpr (MORE2) { store_staged(t + 2); load_staged(t + 3 < steps ? t + 3 : steps - 1, std::true_type()); }
        }
        products(Last(), [&](int a) {
            if constexpr (MORE) if (a == 0) { __builtin_amdgcn_sched_barrier(0); read(t + 1, First(), !MORE2 && ragged); __builtin_amdgcn_sched_barrier(0); }
            if constexpr (DMA && MORE2) {                                           // the first half of the fill behind it
#pragma unroll
                for (int i = a * (QT / 2) / FN; i < (a + 1) * (QT / 2) / FN; i++) fill(t + 2, i);
            }
        });
        __builtin_amdgcn_sched_barrier(0);
    };
    int t = 0;
#pragma unroll 1
    for (; t + 2 < steps; t++) step(t, std::true_type(), std::true_type());
    if (t + 1 < steps) { step(t, std::true_type(), std::false_type()); t++; }
    if (t < steps) step(t, std::false_type(), std::false_type());

    // ---- epilogue: acc[a][b][i] = tile row 32 (wn FN + a) + 8 (i / 4) + 4 g + i % 4 of the weights, slot 32 (wm FM + b) + r.  The fp32 tile goes through LDS (chunks of four columns, xor-ed with the slot) so that a
    // thread stores eight consecutive columns: whole 512-byte rows instead of 8-byte pieces.
    constexpr int PB = 2 * S::STAGE / (BN * 4) / (32 * WM) < FM ? 2 * S::STAGE / (BN * 4) / (32 * WM) : FM;   // slot groups of a wave that fit at once
    const float* bias = p.bias ? p.bias + (long long)tile.e * p.w_rows : nullptr;
#pragma unroll
    for (int b0 = 0; b0 < FM; b0 += PB) {
        __syncthreads();
#pragma unroll
        for (int a = 0; a < FN; a++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int j = (wn * FN + a) * 8 + 2 * q + g;                        // chunk of four columns
                floatx4 m = {1, 1, 1, 1};
                if constexpr (DEQ && XK == SM_F16) m = *(const floatx4*)(wmul + 4 * j);
#pragma unroll
                for (int b = 0; b < PB; b++) {
                    const floatx16 v = acc[a][b0 + b];
                    *(floatx4*)(lds + ((wm * PB + b) * 32 + r) * BN * 4 + ((j ^ (r & 15)) << 4)) = floatx4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]} * m;
                }
            }
        __syncthreads();
        const int per = cols / 8;
        for (int o = tid; o < PB * WM * 32 * per; o += THREADS) {
            const int l = o / per, c = o - l * per, n = n0 + c * 8;                 // LDS row, group of eight columns
            const int slot = (l / (32 * PB) * FM + b0) * 32 + l % (32 * PB);
            if (slot >= tile.rows || n >= p.N) continue;
            const char* row = lds + l * BN * 4;
            const int j = p.gated ? (c >> 1) * 8 + (c & 1) * 2 : 2 * c, x = l & 15;
            float v[8];
            auto get = [&](int ch, float* q, long long up) {
                const floatx4 q0 = *(const floatx4*)(row + ((ch ^ x) << 4)), q1 = *(const floatx4*)(row + (((ch + 1) ^ x) << 4));
#pragma unroll
                for (int i = 0; i < 4; i++) { q[i] = q0[i]; q[4 + i] = q1[i]; }
                if (p.rows && slot_row(slot) < 0) for (int i = 0; i < 8; i++) q[i] = 0.f;
                if (bias) for (int i = 0; i < 8; i++) if (n + i < p.N) q[i] += bias[n + i + up];
            };
            get(j, v, 0);
            if (p.gated) {
                float u[8]; get(j + 4, u, p.N);
                for (int i = 0; i < 8; i++) v[i] = lin_silu(v[i]) * u[i];
            } else if (p.act != SM_ACT_NONE) for (int i = 0; i < 8; i++) v[i] = lin_act(v[i], p.act, p.slope);
            const long long out = (tile.row0 + slot) * p.y_ld + n;
            if (p.y_vec && n + 8 <= p.N) lin_store8(p.y, out, v, p.y_type);
            else for (int i = 0; i < 8; i++) if (n + i < p.N) lin_store1(p.y, out + i, v[i], p.y_type);
        }
    }
}

template <int XK, int WK, int WN, int WM, int FN, int FM, bool DMA> static int lin_tile(const LinearParams& q, hipStream_t s) {
    typedef LinTileShape<XK, WK, WN, WM, FN, FM, DMA> S;
    LinearParams p = q;
    const int cols = p.gated ? S::BN / 2 : S::BN;
    p.n_tiles = (p.N + cols - 1) / cols;
    p.m_tiles = lin_row_tiles(p, S::BM);
    const long long blocks = (p.m_tiles * p.n_tiles + 7) / 8 * 8;
    SM_REQUIRE(blocks < (1ll << 31), "linear: %lld row tiles x %d column tiles exceed one launch", p.m_tiles, p.n_tiles);
    lin_tile_kernel<XK, WK, WN, WM, FN, FM, DMA><<<dim3((unsigned)blocks), S::THREADS, 0, s>>>(p);
    SM_LAUNCH_CHECK();
    return SM_OK;
}
