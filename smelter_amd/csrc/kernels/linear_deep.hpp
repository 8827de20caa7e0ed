// smelter_amd/csrc/kernels/linear_deep.hpp — linear layers on some tens to some hundred rows: small tiles (128 weight rows x 64 or 128 slots, four waves) with several steps of K in flight.
//
// With few tiles a CU waits: for memory (the bytes that it has asked for, over the time they take, are its rate), and for LDS, whose latency is longer than the few products of a phase.  The tile
// kernel asks for one step ahead and reads a quarter of a step ahead; here ST - 1 steps are on their way and the fragments of a whole step are read while the products of the one before run: 512 rows
// of 4096 x 4096 in fp16 take 29 us, 64 rows 17.  That needs every load of the loop to be an LDS-DMA (their completion is counted; a load into registers would make the compiler wait for all of
// them): MX4 weights under a 16-bit x stay packed in LDS (32 bytes a row and step instead of 128) and become 16-bit values behind the fragment read, and the scale bytes of the whole run of K are
// put into LDS once, in front of the loop.  For the packed weights a lane group takes the chunks 4 g .. 4 g + 3 of a row — one MX4 block, one scale — instead of 2 P + g; the order in which k are
// added is free as long as both operands agree.  (Both sides in MX4 gain nothing: their steps are four times as long in K, few, and their scales are a load of their own.)
#pragma once
#include "linear_tile.hpp"
#include <atomic>

template <int N> __device__ __forceinline__ void lin_arrive_n() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

template <int XK, int WK, int FM, int ST> struct LinDeepShape {
    static constexpr int THREADS = 256, BN = 128, BM = 64 * FM;
    static constexpr bool DEQ = WK == SM_MX4;
    static constexpr int WB = DEQ ? 32 : 128, STAGE = BN * WB + BM * 128;          // bytes of a weight row and step
    static constexpr int SROWS = DEQ ? BN : 0;                                      // rows with scales
    static constexpr int pitch(int blocks) { return (((blocks + 15) >> 4) | 1) << 4; }   // scale bytes of a row in LDS: an odd number of 16-byte units, so that rows start in different banks
    static constexpr int DUMP = BN * BM * 4 < 65536 ? BN * BM * 4 : 65536;          // the epilogue's share
    static int lds(int blocks) { const int a = ST * STAGE + SROWS * pitch(blocks) + (DEQ ? BN * 4 : 0); return a > DUMP + BN * 4 ? a : DUMP + BN * 4; }
};

template <int XK, int WK, int FM, int ST> __global__ __launch_bounds__(256) void lin_deep_kernel(LinearParams p, int most) {
    typedef LinDeepShape<XK, WK, FM, ST> S;
    constexpr int FN = 2, BN = S::BN, BM = S::BM;
    constexpr bool DEQ = S::DEQ;
    extern __shared__ __align__(16) char dlds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, g = lane >> 5;
    int split, nt;
    const LinTile tile = lin_pick_tile<false>(p, BM, &split, &nt);
    if (tile.rows == 0) return;
    const int nb = (p.K + 31) >> 5, w_bytes = DEQ ? 16 * nb : 2 * p.K, x_bytes = 2 * p.K;
    const int every = (x_bytes + 127) >> 7, first = (int)((long long)every * split / p.splits), steps = (int)((long long)every * (split + 1) / p.splits);
    constexpr int BS = 2;                                                           // blocks of a step
    const int n0 = nt * (p.gated ? BN / 2 : BN);
    const char* wexp = p.w + tile.e * p.w_es;
    const char* xbase = p.rows ? p.x : p.x + tile.row0 * p.x_ld;

    // ---- LDS-DMA: 64 lanes fill 1 KB: 8 rows of 128 bytes (chunk c of row r at place c ^ (r & 7) ^ (r >> 4 & 1)), or 32 rows of 32 bytes of packed weights
    constexpr int QW = BN * S::WB / 4096, QX = BM / 32, QT = QW + QX;
    unsigned woff[QW], xoff[QX];
    const int wrow = DEQ ? lane >> 1 : lane >> 3, chunk = (lane & 7) ^ (lane >> 3);
    auto swz = [](int row) { return row >> 4 & 1; };
#pragma unroll
    for (int i = 0; i < QW; i++) woff[i] = (unsigned)(lin_weight_row(p, n0, (wave * QW + i) * (DEQ ? 32 : 8) + wrow) * p.w_ld);
#pragma unroll
    for (int i = 0; i < QX; i++) { const long long s = lin_slot_row(p, tile, (wave * QX + i) * 8 + (lane >> 3)); xoff[i] = (unsigned)((s < 0 ? 0 : p.rows ? s : s - tile.row0) * p.x_ld); }
    const unsigned lds0 = lin_lds_addr(dlds);
    auto fill = [&](int t, int slot, int i) {                                       // instruction i of QT of step t; behind the end of a row: its last chunk again
        const unsigned st = lds0 + slot * S::STAGE;
        if (i < QW) {
            int k = DEQ ? t * 32 + (lane & 1) * 16 : t * 128 + (chunk ^ swz((wave * QW + i) * 8)) * 16; if (k > w_bytes - 16) k = w_bytes - 16;
            lin_dma16(wexp, woff[i < QW ? i : 0] + k, st + (wave * QW + i) * 1024);
        } else {
            int k = t * 128 + (chunk ^ swz((wave * QX + i - QW) * 8)) * 16; if (k > x_bytes - 16) k = x_bytes - 16;
            lin_dma16(xbase, xoff[i < QW ? 0 : i - QW] + k, st + BN * S::WB + (wave * QX + i - QW) * 1024);
        }
    };
    const int ahead = steps - first < ST ? steps - first : ST;
    for (int t = 0; t < ahead; t++) {
#pragma unroll
        for (int i = 0; i < QT; i++) fill(first + t, t, i);
    }

    // ---- scales of the run: blocks b0 .. b0 + blocks - 1 of each row
    const int b0 = first * BS, blocks = (steps * BS < nb ? steps * BS : nb) - b0, pitch = S::pitch(most);
    unsigned char* scale = (unsigned char*)dlds + ST * S::STAGE;
    float* wmul = (float*)(dlds + (ST * S::STAGE + S::SROWS * pitch > S::DUMP ? ST * S::STAGE + S::SROWS * pitch : S::DUMP));
    if constexpr (DEQ) {
        const int groups = (blocks + 15) >> 4;
        for (int o = tid; o < S::SROWS * groups; o += 256) {
            const int j = o / groups, q = o - j * groups, at = b0 + 16 * q;
            const unsigned char* src = p.ws + tile.e * p.ws_es + lin_weight_row(p, n0, j) * p.ws_ld;
            intx4_t v;
            if (at + 16 <= nb) __builtin_memcpy(&v, src + at, 16);
            else {                                                                  // behind the end of the row (codes 0): its last scale again
                unsigned c[4] = {0, 0, 0, 0};
#pragma unroll
                for (int b = 0; b < 16; b++) c[b >> 2] |= (unsigned)src[at + b < nb ? at + b : nb - 1] << (8 * (b & 3));
                v = intx4_t{(int)c[0], (int)c[1], (int)c[2], (int)c[3]};
            }
            *(intx4_t*)(scale + j * pitch + 16 * q) = v;
        }
        if constexpr (XK == SM_F16) {                                               // relative to the row's largest scale of the run; a row that reaches too far is marked by a negative factor
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            const int j = tid >> 1;
            unsigned char* row = scale + j * pitch;
            unsigned* words = (unsigned*)row;                                        // (what lies behind the run's last block are scales too)
            const int count = (blocks + 3) >> 2;
            LinSpread all;
            for (int q = tid & 1; q < count; q += 2) all.look(words[q]);
            int top = all.top(), low = all.low();
            int o = __shfl_xor(top, 1); top = top > o ? top : o;
            o = __shfl_xor(low, 1); low = low < o ? low : o;
            const bool nan = top == 255;                                             // a NaN block: the largest of the others, its own byte stays
            if (nan) { top = 0; for (int b = 0; b < blocks; b++) top = lin_top_of(top, row[b]); }
            if (top < 14) top = 14;
            int far = 0;
            if (top - low > LIN_REACH) {
                const char* codes = wexp + lin_weight_row(p, n0, j) * p.w_ld + 16ll * b0;
                for (int b = tid & 1; b < blocks; b += 2)
                    if (lin_relative(row[b], top) < 140 - LIN_REACH) { intx4_t c; __builtin_memcpy(&c, codes + 16ll * b, 16); far |= (c[0] | c[1] | c[2] | c[3]) & 0x77777777; }
            }
            __builtin_amdgcn_wave_barrier();                                         // (the two threads of a row have read all of it)
            const ushortx2_t up = {140, 140}, down = {(unsigned short)top, (unsigned short)top};
            for (int q = tid & 1; q < count; q += 2) {
                const unsigned v = words[q];
                if (nan) { for (int i = 0; i < 4; i++) row[4 * q + i] = lin_relative(v >> (8 * i) & 255, top); }
                else {
                    const ushortx2_t a = __builtin_bit_cast(ushortx2_t, v & 0x00ff00ffu) + up, b = __builtin_bit_cast(ushortx2_t, v >> 8 & 0x00ff00ffu) + up;
                    words[q] = __builtin_bit_cast(unsigned, __builtin_elementwise_sub_sat(a, down)) | __builtin_bit_cast(unsigned, __builtin_elementwise_sub_sat(b, down)) << 8;
                }
            }
            far |= __shfl_xor(far, 1);
            if (!(tid & 1)) wmul[j] = far ? -1.f : lin_top_scale(top);
        }
    }

    const int wn = wave & 1, wm = wave >> 1;
    floatx16 acc[FN][FM];
#pragma unroll
    for (int a = 0; a < FN; a++)
#pragma unroll
        for (int b = 0; b < FM; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[a][b][i] = 0.f;
    // two sets of a whole step's fragments: while the products of one run, the other is read
    constexpr int NW = DEQ ? 1 : 4;                                                 // (packed weights: all four phases of a row in one read, one scale)
    intx4_t wf[2][FN][NW], xf[2][FM][4]; int wsc[2][FN];
    auto read = [&](int t, int slot, auto set, bool masked) {
        constexpr int B = decltype(set)::value;
        const char* st = dlds + slot * S::STAGE + r * S::WB;
        const char* sx = dlds + slot * S::STAGE + BN * S::WB + r * 128;
        if constexpr (DEQ) {
            const int q = 2 * t + g - b0;
#pragma unroll
            for (int a = 0; a < FN; a++) {
                wf[B][a][0] = *(const intx4_t*)(st + (wn * FN + a) * 32 * S::WB + g * 16);
                wsc[B][a] = scale[((wn * FN + a) * 32 + r) * pitch + (q < blocks ? q : blocks - 1)];
                if (masked && q >= blocks) wsc[B][a] = 0;                           // (behind the end: finite, under zeros of x)
            }
        }
#pragma unroll
        for (int P = 0; P < 4; P++) {
            const int ch = DEQ ? 4 * g + P : 2 * P + g, at = (ch ^ (lane & 7) ^ swz(r)) << 4;
            if constexpr (!DEQ) {
#pragma unroll
                for (int a = 0; a < FN; a++) wf[B][a][P] = *(const intx4_t*)(st + (wn * FN + a) * 32 * S::WB + at);
            }
#pragma unroll
            for (int b = 0; b < FM; b++) xf[B][b][P] = *(const intx4_t*)(sx + (wm * FM + b) * 32 * 128 + at);
            if (masked) {                                                           // chunks behind the end of the row
                const bool dead = t * 128 + ch * 16 >= x_bytes;
                if constexpr (!DEQ) {
#pragma unroll
                    for (int a = 0; a < FN; a++) wf[B][a][P] = dead ? intx4_t{0, 0, 0, 0} : wf[B][a][P];
                }
#pragma unroll
                for (int b = 0; b < FM; b++) xf[B][b][P] = dead ? intx4_t{0, 0, 0, 0} : xf[B][b][P];
            }
        }
    };
    const bool ragged = (x_bytes & 127) && steps == every;
    typedef std::integral_constant<int, 0> I0; typedef std::integral_constant<int, 1> I1;
    int slot = 0;
    // FULL: steps t + 2 .. t + ST - 1 have been asked for, and step t + ST exists
    auto step = [&](int t, auto set, auto has_next, auto full) {
        constexpr int B = decltype(set)::value;
        constexpr bool MORE = decltype(has_next)::value, FULL = decltype(full)::value;
        const int next = slot + 1 == ST ? 0 : slot + 1;
        if constexpr (MORE) {
            lin_arrive_n<FULL ? (ST - 2) * QT : 0>();                               // step t + 1 is in LDS for everybody; everybody has read the whole of step t
            read(t + 1, next, std::integral_constant<int, 1 - B>(), !FULL && ragged && t + 2 == steps);
            __builtin_amdgcn_sched_barrier(0);
        }
        sm_static_for<0, 4>([&](auto phase) {
            constexpr int P = decltype(phase)::value;
#pragma unroll
            for (int a = 0; a < FN; a++) {
                intx4_t w;
                if constexpr (DEQ) w = mx4_to16<XK>(wf[B][a][0][P], mx4_scale(wsc[B][a])); else w = wf[B][a][P];
#pragma unroll
                for (int b = 0; b < FM; b++) acc[a][b] = lin_mma16<XK>(w, xf[B][b][P], acc[a][b]);
            }
            if constexpr (FULL) {
#pragma unroll
                for (int i = P * QT / 4; i < (P + 1) * QT / 4; i++) fill(t + ST, slot, i);
            }
        });
        __builtin_amdgcn_sched_barrier(0);
        slot = next;
    };
    auto tail = [&](int t, auto set) {
        if (t + ST < steps) step(t, set, std::true_type(), std::true_type());
        else if (t + 1 < steps) step(t, set, std::true_type(), std::false_type());
        else step(t, set, std::false_type(), std::false_type());
    };
    if (steps > first) {
        if (ahead == ST) lin_arrive_n<(ST - 1) * QT>(); else lin_arrive_n<0>();
        int t = first;
        if constexpr (DEQ && XK == SM_F16) {
            if (__any(wmul[lane] < 0.f || wmul[64 + lane] < 0.f)) {                 // (every wave sees the same)
                lin_arrive_n<0>();
                if (tid < BN) wmul[tid] = 1.f;
                const char* xr[FM]; int xk[FM];
#pragma unroll
                for (int b = 0; b < FM; b++) { const long long row = lin_slot_row(p, tile, 32 * (wm * FM + b) + r); xr[b] = p.x + (row < 0 ? 0 : row) * p.x_ld; xk[b] = row < 0 ? 0 : p.K; }
#pragma unroll
                for (int a = 0; a < FN; a++) {
                    const long long row = lin_weight_row(p, n0, 32 * (wn * FN + a) + r);
                    lin_exact_blocks<32, FM>(wexp + row * p.w_ld, p.ws + tile.e * p.ws_es + row * p.ws_ld, xr, xk, b0, b0 + blocks,
                                             [&](int b, intx4_t w, intx4_t x) { acc[a][b] = lin_mma16<SM_BF16>(w, x, acc[a][b]); },
                                             [&] {
#pragma unroll
                                                 for (int b = 0; b < FM; b++) acc[a][b] = acc[a][b] * 0x1p64f * 0x1p64f;
                                             });
                }
                t = steps;
            }
        }
        if (t < steps) read(first, 0, I0(), ragged && steps == first + 1);
#pragma unroll 1
        for (; t + 1 + ST < steps; t += 2) { step(t, I0(), std::true_type(), std::true_type()); step(t + 1, I1(), std::true_type(), std::true_type()); }
#pragma unroll 1
        for (; t < steps; t += 2) { tail(t, I0()); if (t + 1 < steps) tail(t + 1, I1()); }
    }
    lin_finish<XK, 32, 2, 2, FN, FM, S::DUMP, DEQ && XK == SM_F16>(p, tile, split, n0, acc, dlds, wmul);
}

// a kernel's dynamic LDS may be the whole 160 KB on the current device; asked for once per kernel and device
template <class Tag> static int lin_allow_lds_once(const void* kernel) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    SM_HIP_CHECK(hipGetDevice(&dev));
    if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return SM_OK;
    SM_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return SM_OK;
}
template <int XK, int WK, int FM, int ST> static bool lin_deep_fits(const LinearParams& p) {
    typedef LinDeepShape<XK, WK, FM, ST> S;
    const int every = (int)((2ll * p.K + 127) / 128), most = (every + p.splits - 1) / p.splits * 2;
    return S::lds(most) <= 160 * 1024;
}
template <int XK, int WK, int FM, int ST> static int lin_deep(const LinearParams& q, hipStream_t s) {
    typedef LinDeepShape<XK, WK, FM, ST> S;
    LinearParams p = q;
    const int cols = p.gated ? S::BN / 2 : S::BN;
    p.n_tiles = (p.N + cols - 1) / cols;
    p.m_tiles = lin_row_tiles(p, S::BM);
    const long long blocks = (p.m_tiles * p.n_tiles + 7) / 8 * 8 * p.splits;
    SM_REQUIRE(lin_one_launch(blocks, S::THREADS), "linear: %lld row tiles x %d column tiles exceed one launch", p.m_tiles, p.n_tiles);
    const int every = (int)((2ll * p.K + 127) / 128), most = (every + p.splits - 1) / p.splits * 2;
    const auto kernel = lin_deep_kernel<XK, WK, FM, ST>;
    if (int rc = lin_allow_lds_once<S>((const void*)kernel)) return rc;
    kernel<<<dim3((unsigned)blocks), S::THREADS, S::lds(most), s>>>(p, most);
    SM_LAUNCH_CHECK();
    return SM_OK;
}
