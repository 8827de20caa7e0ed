// smelter_amd/csrc/kernels/linear.hip — linear layers with 16-bit or MX4 weights, dense or grouped by expert: argument checks and the choice of kernel.
#include "linear_stream.hpp"

template <int XK, int WK, int NB> static int lin_stream_nb(LinearParams p, hipStream_t s) {
    const int cols = p.gated ? 8 * NB : 16 * NB;
    p.n_tiles = (p.N + cols - 1) / cols;
    p.m_tiles = lin_row_tiles(p, 16);
    const long long blocks = p.m_tiles * p.n_tiles;
    const int chunks = ((p.K + 31) / 32 + (WK == SM_MX4 ? 15 : 3)) / (WK == SM_MX4 ? 16 : 4);
    int waves = blocks >= 4 * SM_NUM_CU ? 4 : 8;                                    // many blocks: fewer sums to join (16 experts bf16 2048 x 2048: 13.2 us with 4 waves, 15.4 with 8; one 4096 x 4096: 15.0, 13.6)
    while (waves > 1 && waves > chunks) waves /= 2;
    SM_REQUIRE(lin_one_launch(blocks, 64 * waves), "linear: %lld row tiles x %d column tiles exceed one launch", p.m_tiles, p.n_tiles);
    lin_stream_kernel<XK, WK, NB><<<dim3((unsigned)blocks), 64 * waves, (size_t)waves * NB * 16 * 17 * 4, s>>>(p);
    SM_LAUNCH_CHECK();
    return SM_OK;
}
// four groups of weight rows for a wave where that leaves a block for every CU (64 experts 8192 x 2048 MX4: 77 us against 89), two otherwise (4096 x 4096: 7.7 against 10.6)
template <int XK, int WK> static int lin_stream(const LinearParams& p, hipStream_t s) {
    const long long tiles = lin_row_tiles(p, 16) * ((p.w_rows + 63) / 64);
    return tiles >= SM_NUM_CU ? lin_stream_nb<XK, WK, 4>(p, s) : lin_stream_nb<XK, WK, 2>(p, s);
}

static int lin_size(int kind, long long K, long long* row, long long* scale_row) {
    if (kind == SM_MX4) { *row = (K + 31) / 32 * 16; *scale_row = (K + 31) / 32; } else { *row = (kind == SM_F32 ? 4 : 2) * K; *scale_row = 0; }
    return 0;
}

struct LinearPlan { int shape, splits, deep; };                                      // shape -1: the streaming kernel
static long long lin_part_ld(long long w_rows) { return (w_rows + 3) / 4 * 4; }

// Which kernel, by sizes alone (the offsets are on the device): `per` = slots of an average group.
static LinearPlan lin_plan(const sm_linear_desc* d, bool grouped, bool gathered) {
    LinearParams p = {};
    long long xr, xsr, wr, wsr;
    lin_size(d->x_type, d->K, &xr, &xsr); lin_size(d->w_type, d->K, &wr, &wsr);
    p.M = d->M; p.T = d->T; p.N = d->N; p.E = d->E; p.gated = d->gated != 0;
    p.offsets = grouped ? (const int*)8 : nullptr; p.rows = gathered ? (const int*)8 : nullptr;     // (looked at for being there only)
    p.x_ld = d->x_type != SM_MX4 && d->x_ld ? 2 * d->x_ld : xr; p.w_es = wr * (p.gated ? 2 : 1) * d->N;
    const long long per = grouped ? (d->M + d->E - 1) / d->E : d->M;
    LinearPlan plan = {-1, 1, 0};
    if (per <= 16 || d->K < 8 || !lin_tile_fits(p)) return plan;
    // the tiles to expect: groups end anywhere inside their last tile (E = 1: of all slots)
    auto tiles = [&](int bn, int bm) {
        const int cols = p.gated ? bn / 2 : bn;
        const long long groups = d->M < d->E ? d->M : d->E, most = lin_row_tiles(p, bm), half = d->M / bm + (groups + 1) / 2, row = half < groups ? groups : half;
        return (groups == 1 || row > most ? most : row) * ((p.N + cols - 1) / cols);
    };
    // Times in units of a round of 512 tiles of 128 x 128, two on a CU (69 us of fp16 with K = 4096, 29 of MX4 by MX4).  A round that is not full costs less, but not in proportion, and differently
    // for each tile: a CU that holds one tile of 128 x 128 needs 0.6 of the time it needs for two.  Measured on 4096 x 4096 weights in fp16 (us; tiles of 128 x 128 / 256 x 256 / 128 x 64):
    // 512 rows 39 / 60 / 29, 640 rows 40 / 60 / 44, 1280 rows 55 / 61 / 56, 2048 rows 69 / 67 / 98, 2304 rows 109 / 80 / 101, 4096 rows 135 / 108 / 168; MX4 weights under them: 42 / 88 / 32,
    // 43 / 87 / 52, 59 / 88 / 73, 79 / 91 / 127, 131 / 91 / 130, 152 / 109 / 218.
    const long long n0 = tiles(128, 128), n1 = tiles(256, 256), n2 = tiles(128, 64);
    const bool w16 = d->w_type != SM_MX4;
    auto time = [&](int shape, long long n) {
        const long long round = shape == 0 ? 512 : shape == 1 ? 256 : 768, r = n % round;
        const double full = shape == 0 ? 0.97 : shape == 1 ? (w16 ? 1.55 : 1.38) : 0.95;
        const double part = r == 0 ? 0 : shape == 0 ? (r <= 256 ? 0.6 : 0.8 + 0.2 * (r - 256) / 256) : shape == 1 ? (w16 && r <= 128 ? 0.9 : r <= 192 ? 1.1 : full)    // (w16: the halves of lin_pick_tile)
                          : r <= 256 ? 0.42 : r <= 512 ? 0.7 : w16 ? 0.82 : 0.95;
        return n / round * full + part;
    };
    // the number of tiles of ragged groups may lie on either side of a whole round: the mean over a tenth more and less
    auto mean = [&](int shape, long long n) { return !grouped || d->E == 1 ? time(shape, n) : (time(shape, n - n / 10) + time(shape, n) + time(shape, n + n / 10)) / 3; };
    const double t0 = mean(0, n0), t1 = mean(1, n1), t2 = mean(2, n2);
    plan.shape = t2 <= t0 && t2 <= t1 ? 2 : t0 <= t1 ? 0 : 1;
    const long long n = plan.shape == 2 ? n2 : n0;
    plan.deep = d->x_type != SM_MX4 && plan.shape != 1 && n <= SM_NUM_CU;
    if (plan.shape == 2 && n * 2 <= SM_NUM_CU && d->E <= 64) {
        // Runs of K, as many as fill the card: a step of a block that is alone on its CU takes 0.3 us (MX4 by MX4, four times as long a piece of K: 0.55), the sums go to memory and back, the
        // joining launch costs 3.5 us.  bf16, us with 1 / 2 / 4 / 8 runs: 64 rows of 2048 x 8192 42 / 29 / 21 / 18, 100 rows of 4096 x 4096 25 / 22 / 18.5 / 26, 64 rows of 8192 x 2048 16.7 / 17.7 /
        // 18.3 / 25.8; MX4 by MX4: 100 rows of 8192 x 8192 25.6 / 23.2 / 22 / 29, of 4096 x 4096 11.8 / 13.9 / 14.1.
        const int steps = (int)(((d->x_type == SM_MX4 ? xr : 2ll * d->K) + 127) / 128);
        const double step = d->x_type == SM_MX4 ? 0.55 : 0.3, sums = d->M * (double)d->N * (d->gated ? 2 : 1) * 8 / 4e6;
        double best = steps * step;
        for (int s = 2; s <= 8 && s * n <= SM_NUM_CU && s <= steps / 4; s++) {
            const double t = (steps + s - 1) / s * step + 3.5 + s * sums;
            if (t < best) { best = t; plan.splits = s; }
        }
    }
    return plan;
}

// fp32 rows: each becomes several 16-bit ones that add up to it, the product runs on all of them — the weights are read once — and lin_join_kernel adds their sums, bias and activation.
// bf16 (under bf16 and MX4 weights): three parts of eight bits, each cut, not rounded: all 24 bits, and no part is infinite where the value is not.
// fp16 (under fp16 weights): fp16 ends at 65504 and holds nothing below 2^-24, so a row is first scaled by a power of two that puts its largest value at 2^15 .. 2^16; then three parts, 2^-11 apart,
// each cut (not rounded), so that none passes 65504.  They hold all 24 bits of every value down to 2^-38 of the largest.  A row with smaller ones, an infinity or a NaN is marked: its parts are zero,
// the join leaves it out, and lin_stream_kernel multiplies it in fp32 (one launch more, 4 us where no row is marked).  4096 rows of 4096 x 4096: 523 us, 1870 where all are marked.
// 192 slots on 32 experts of 2048 x 1024 in MX4: 29 us (three launches) against 13 of bf16 rows; 4096 rows of 4096 x 4096: 464.
__device__ __forceinline__ floatx4 lin_load4(const float* row, int k, int K) {       // zero behind the row's end
    floatx4 v = {0, 0, 0, 0};
    if (k + 4 <= K) __builtin_memcpy(&v, row + k, 16);
    else for (int q = 0; q < 3; q++) if (k + q < K) v[q] = row[k + q];
    return v;
}
#define LIN_PARTS 3
template <class H> __global__ __launch_bounds__(256) void lin_parts_kernel(const float* x, long long x_ld, const int* offsets, const int* rows, long long M, long long T, int K, int E, H* out, long long ld,
                                                                           int* more, int* power) {
    constexpr int PARTS = LIN_PARTS;
    constexpr bool SCALED = std::is_same_v<H, half_t>;
    if (offsets && blockIdx.x == 0) for (int e = threadIdx.x; e <= E; e += blockDim.x) more[e] = (int)(PARTS * lin_clamp(offsets[e], M));
    __shared__ unsigned ends[2][4];                                                  // largest magnitude, smallest one that is not 0, of the waves
    for (long long s = blockIdx.x; s < M; s += gridDim.x) {                          // a block to a slot
        const long long r = rows ? rows[s] : s;
        const bool live = r >= 0 && r < T;
        const float* src = x + (live ? r : 0) * x_ld;
        int up = 0; bool marked = false;
        if constexpr (SCALED) {
            unsigned hi = 0, lo = ~0u;
            for (int k = 4 * threadIdx.x; k < K && live; k += 1024) {
                const floatx4 v = lin_load4(src, k, K);
#pragma unroll
                for (int q = 0; q < 4; q++) { const float f = v[q] /* (__builtin_bit_cast of a vector element takes the first) */; const unsigned b = __builtin_bit_cast(unsigned, f) & 0x7fffffffu; hi = hi > b ? hi : b; if (b) lo = lo < b ? lo : b; }
            }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) { const unsigned a = __shfl_xor(hi, d), c = __shfl_xor(lo, d); hi = hi > a ? hi : a; lo = lo < c ? lo : c; }
            __syncthreads();                                                         // (of the slot before)
            if ((threadIdx.x & 63) == 0) { ends[0][threadIdx.x >> 6] = hi; ends[1][threadIdx.x >> 6] = lo; }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 4; w++) { const unsigned a = ends[0][w], c = ends[1][w]; hi = hi > a ? hi : a; lo = lo < c ? lo : c; }
            if (hi) {
                up = 16 - __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, hi));    // |v| < 2^(16 - up)
                marked = hi >= 0x7f800000u || ldexpf(__builtin_bit_cast(float, lo), up) < 0x1p-23f;
            }
            if (threadIdx.x == 0) power[s] = marked ? LIN_MARKED : -up;
        }
        H* to = out + PARTS * s * ld;
        typedef H H4 __attribute__((ext_vector_type(4)));
        for (int k = 4 * threadIdx.x; k < K; k += 1024) {                           // (rows of the parts end behind a whole quad)
            floatx4 v = {0, 0, 0, 0};
            if (live && !marked) v = lin_load4(src, k, K);
            H4 h[PARTS];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if constexpr (SCALED) {
                    float left = ldexpf(v[q], up);
#pragma unroll
                    for (int i = 0; i < PARTS; i++) { h[i][q] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(left, left))[0]; left = (left - (float)h[i][q]) * 0x1p11f; }
                } else {
                    float left = v[q];
#pragma unroll
                    for (int i = 0; i < PARTS; i++) {
                        const bool fine = __builtin_fabsf(left) < __builtin_inff();
                        h[i][q] = fine ? (H)__builtin_bit_cast(float, __builtin_bit_cast(unsigned, left) & 0xffff0000u) : (H)left;
                        left = fine ? left - (float)h[i][q] : 0.f;                   // (an infinity, a NaN: once)
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < PARTS; i++) *(H4*)(to + i * ld + k) = h[i];
        }
    }
}
struct LinearParts { sm_linear_desc in; size_t more, power, sums, inner, total; };   // the product on the parts of every row; where its offsets, the rows' powers of two, its sums and its own workspace lie behind them
static LinearParts lin_parts(const sm_linear_desc* d, bool grouped) {
    LinearParts a; a.in = *d;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const bool scaled = d->w_type == SM_F16;
    a.in.M = a.in.T = LIN_PARTS * d->M; a.in.N = d->gated ? 2 * d->N : d->N; a.in.gated = 0; a.in.act = SM_ACT_NONE;
    a.in.x_type = scaled ? SM_F16 : SM_BF16; a.in.y_type = SM_F32; a.in.x_ld = (d->K + 7ll) / 8 * 8; a.in.y_ld = lin_part_ld(a.in.N);
    a.more = up((size_t)a.in.M * a.in.x_ld * 2); a.power = a.more + up(grouped ? (d->E + 1ll) * 4 : 0); a.sums = a.power + up(scaled ? (size_t)d->M * 4 : 0);
    a.inner = a.sums + up((size_t)a.in.M * a.in.y_ld * 4);
    a.total = a.inner + sm_linear_workspace_bytes(&a.in, grouped, 0);
    return a;
}

extern "C" size_t sm_linear_workspace_bytes(const sm_linear_desc* d, int32_t grouped, int32_t gathered) {
    if (!d || d->M <= 0 || d->N <= 0 || d->E < 1 || d->K < 0) return 0;
    if (d->x_type == SM_F32) return lin_parts(d, grouped).total;
    const LinearPlan plan = lin_plan(d, grouped, gathered);
    return plan.shape < 0 || plan.splits <= 1 ? 0 : (size_t)plan.splits * d->M * lin_part_ld((d->gated ? 2ll : 1ll) * d->N) * 4;
}

extern "C" int sm_linear_fwd(const sm_linear_desc* d, const void* x, const void* x_scales, const void* w, const void* w_scales, const float* bias, const int32_t* offsets,
                             const int32_t* rows, void* y, void* workspace, size_t workspace_bytes, sm_stream_t stream) {
    SM_REQUIRE(d, "linear: null descriptor");
    SM_REQUIRE(d->M >= 0 && d->T >= 0 && d->N >= 0 && d->K >= 0 && d->E >= 1, "linear: sizes M %lld, T %lld, N %d, K %d, E %d", (long long)d->M, (long long)d->T, d->N, d->K, d->E);
    SM_REQUIRE(d->N <= (1 << 29) && d->K <= (1 << 29) && d->M < (1ll << 31) && d->T < (1ll << 31) && d->E <= (1 << 20), "linear: a size beyond what the kernels index");
    const bool x16 = d->x_type == SM_F16 || d->x_type == SM_BF16;
    const bool x32 = d->x_type == SM_F32, w16 = d->w_type == SM_F16 || d->w_type == SM_BF16;
    SM_REQUIRE((x16 && (d->w_type == d->x_type || d->w_type == SM_MX4)) || (d->x_type == SM_MX4 && d->w_type == SM_MX4) || (x32 && (w16 || d->w_type == SM_MX4)),
               "linear: x of type %d on weights of type %d (taken: fp16 or bf16 on weights of the same type or MX4, fp32 on any of them, MX4 on MX4)", d->x_type, d->w_type);
    SM_REQUIRE(d->y_type == SM_F32 || ((d->y_type == SM_F16 || d->y_type == SM_BF16) && (!x16 || d->y_type == SM_F16 || d->y_type == d->x_type)),
               "linear: output type %d for x of type %d (taken: x's own 16-bit type, fp16 or fp32; any of the three for an MX4 x)", d->y_type, d->x_type);
    SM_REQUIRE(d->act >= SM_ACT_NONE && d->act <= SM_ACT_CLIP, "linear: unknown activation %d", d->act);
    SM_REQUIRE(!d->gated || d->act == SM_ACT_NONE, "linear: a gated layer takes no further activation");
    SM_REQUIRE(offsets || d->E == 1, "linear: %d experts without offsets", d->E);
    SM_REQUIRE(rows || d->T >= d->M, "linear: %lld slots on %lld rows of x without a row list", (long long)d->M, (long long)d->T);
    if (d->M == 0 || d->N == 0) return SM_OK;
    LinearParams p = {};
    long long xr, xsr, wr, wsr;
    lin_size(d->x_type, d->K, &xr, &xsr); lin_size(d->w_type, d->K, &wr, &wsr);
    SM_REQUIRE(y, "linear: null output");
    SM_REQUIRE(d->K == 0 || d->T == 0 || (x && w && (d->x_type != SM_MX4 || x_scales) && (d->w_type != SM_MX4 || w_scales)), "linear: null operand");
    p.x = (const char*)x; p.xs = (const unsigned char*)x_scales; p.w = (const char*)w; p.ws = (const unsigned char*)w_scales; p.bias = bias; p.y = y; p.offsets = offsets; p.rows = rows;
    p.M = d->M; p.T = d->T; p.N = d->N; p.K = d->T == 0 ? 0 : d->K; p.E = d->E; p.splits = 1; p.act = d->act; p.slope = d->slope; p.gated = d->gated != 0; p.y_type = d->y_type;
    p.w_rows = p.gated ? 2 * p.N : p.N;
    p.x_ld = d->x_type != SM_MX4 && d->x_ld ? (x32 ? 4 : 2) * d->x_ld : xr; p.xs_ld = xsr; p.w_ld = wr; p.ws_ld = wsr; p.w_es = wr * p.w_rows; p.ws_es = wsr * p.w_rows; p.y_ld = d->y_ld ? d->y_ld : d->N;
    SM_REQUIRE(d->T <= 1 || p.x_ld >= xr, "linear: row stride of x %lld below its %d columns", (long long)d->x_ld, d->K);
    SM_REQUIRE(d->M == 1 || p.y_ld >= d->N, "linear: row stride of y %lld below its %d columns", p.y_ld, d->N);
    const int ye = d->y_type == SM_F32 ? 4 : 2;
    SM_REQUIRE((size_t)y % ye == 0 && (size_t)bias % 4 == 0 && (size_t)offsets % 4 == 0 && (size_t)rows % 4 == 0 && (d->x_type == SM_MX4 || (size_t)x % (x32 ? 4 : 2) == 0) && (d->w_type == SM_MX4 || (size_t)w % 2 == 0),
               "linear: an operand is not aligned to its element");
    SM_REQUIRE((d->x_type != SM_MX4 || (size_t)x % 16 == 0) && (d->w_type != SM_MX4 || (size_t)w % 16 == 0), "linear: MX4 codes need 16-byte alignment");
    p.y_vec = (size_t)y % 16 == 0 && p.y_ld * ye % 16 == 0;
    hipStream_t s = sm_s(stream);
    if (x32) {
        SM_REQUIRE(d->M < (1ll << 31) / LIN_PARTS && d->M * ((d->N + 3ll) / 4) < (1ll << 31), "linear: %lld x %d outputs of fp32 rows exceed one launch", (long long)d->M, d->N);
        const LinearParts a = lin_parts(d, offsets != nullptr);
        SM_REQUIRE(workspace && (size_t)workspace % 256 == 0 && workspace_bytes >= a.total, "linear: workspace of %zu bytes (256-byte aligned), %zu wanted", workspace_bytes, a.total);
        char* at = (char*)workspace;
        int* more = offsets ? (int*)(at + a.more) : nullptr;
        int* power = a.in.x_type == SM_F16 ? (int*)(at + a.power) : nullptr;
        const dim3 grid((unsigned)(d->M < SM_NUM_CU * 64 ? d->M : SM_NUM_CU * 64));
        if (power) lin_parts_kernel<half_t><<<grid, 256, 0, s>>>((const float*)x, p.x_ld / 4, offsets, rows, d->M, d->T, p.K, d->E, (half_t*)at, a.in.x_ld, more, power);
        else lin_parts_kernel<bf16_t><<<grid, 256, 0, s>>>((const float*)x, p.x_ld / 4, offsets, rows, d->M, d->T, p.K, d->E, (bf16_t*)at, a.in.x_ld, more, nullptr);
        SM_LAUNCH_CHECK();
        sm_linear_desc in = a.in; in.K = p.K;                                        // (without a row of x nothing of w is read)
        if (int rc = sm_linear_fwd(&in, at, nullptr, w, w_scales, nullptr, more, nullptr, at + a.sums, at + a.inner, workspace_bytes - a.inner, stream)) return rc;
        LinearParams j = p;
        j.part = (float*)(at + a.sums); j.part_ld = a.in.y_ld; j.splits = j.parts = LIN_PARTS; j.power = power;
        if (int rc = lin_join_launch(j, s)) return rc;
        p.power = power;
        return power ? lin_stream<SM_F32, SM_F16>(p, s) : SM_OK;
    }
    LinearPlan plan = lin_plan(d, offsets != nullptr, rows != nullptr);
    if (plan.shape >= 0) {
        const bool dma = d->x_type == SM_MX4 || (p.K % 8 == 0 && (size_t)x % 16 == 0 && p.x_ld % 16 == 0 && (d->w_type == SM_MX4 || (size_t)w % 16 == 0));
        p.splits = plan.splits;
        if (p.splits > 1) {
            p.part_ld = lin_part_ld(p.w_rows);
            SM_REQUIRE(workspace && (size_t)workspace % 16 == 0 && workspace_bytes >= (size_t)p.splits * p.M * p.part_ld * 4, "linear: workspace of %zu bytes (16-byte aligned), %zu wanted", workspace_bytes,
                       (size_t)p.splits * p.M * p.part_ld * 4);
            p.part = (float*)workspace;
        }
        int rc = 1;
        if (dma && plan.deep) rc = lin_deep_launch(p, d->x_type, d->w_type, plan.shape, s);
        if (rc > 0) rc = lin_tile_launch(p, d->x_type, d->w_type, plan.shape, dma, s);
        return rc != SM_OK || p.splits == 1 ? rc : lin_join_launch(p, s);
    }
    if (d->x_type == SM_MX4) return lin_stream<SM_MX4, SM_MX4>(p, s);
    if (d->w_type == SM_MX4) return d->x_type == SM_F16 ? lin_stream<SM_F16, SM_MX4>(p, s) : lin_stream<SM_BF16, SM_MX4>(p, s);
    return d->x_type == SM_F16 ? lin_stream<SM_F16, SM_F16>(p, s) : lin_stream<SM_BF16, SM_BF16>(p, s);
}
