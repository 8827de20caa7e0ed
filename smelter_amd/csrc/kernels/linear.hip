// smelter_amd/csrc/kernels/linear.hip — linear layers with 16-bit or MX4 weights, dense or grouped by expert: argument checks and the choice of kernel.
#include "linear_stream.hpp"

template <int XK, int WK> static int lin_stream(const LinearParams& q, hipStream_t s, int waves) {
    LinearParams p = q;
    const int cols = p.gated ? 16 : 32;
    p.n_tiles = (p.N + cols - 1) / cols;
    const long long per = p.offsets ? (p.M + p.E - 1) / p.E : p.M;      // rows of an average group
    const int mt = per <= 16 ? 1 : per <= 32 ? 2 : 4;
    p.m_tiles = lin_row_tiles(p, 16 * mt);
    const long long blocks = p.m_tiles * p.n_tiles;
    SM_REQUIRE(blocks < (1ll << 31), "linear: %lld row tiles x %d column tiles exceed one launch", p.m_tiles, p.n_tiles);
    if (mt == 4 && waves > 8) waves = 8;
    const size_t lds = (size_t)waves * 2 * mt * 16 * 17 * 4;
    const dim3 grid((unsigned)blocks), block(64 * waves);
    if (mt == 1) lin_stream_kernel<XK, WK, 1><<<grid, block, lds, s>>>(p);
    else if (mt == 2) lin_stream_kernel<XK, WK, 2><<<grid, block, lds, s>>>(p);
    else lin_stream_kernel<XK, WK, 4><<<grid, block, lds, s>>>(p);
    SM_LAUNCH_CHECK();
    return SM_OK;
}

static int lin_size(int kind, long long K, long long* row, long long* scale_row) {
    if (kind == SM_MX4) { *row = (K + 31) / 32 * 16; *scale_row = (K + 31) / 32; } else { *row = 2 * K; *scale_row = 0; }
    return 0;
}

extern "C" int sm_linear_fwd(const sm_linear_desc* d, const void* x, const void* x_scales, const void* w, const void* w_scales, const float* bias, const int32_t* offsets,
                             const int32_t* rows, void* y, sm_stream_t stream) {
    SM_REQUIRE(d, "linear: null descriptor");
    SM_REQUIRE(d->M >= 0 && d->T >= 0 && d->N >= 0 && d->K >= 0 && d->E >= 1, "linear: sizes M %lld, T %lld, N %d, K %d, E %d", (long long)d->M, (long long)d->T, d->N, d->K, d->E);
    SM_REQUIRE(d->N <= (1 << 29) && d->K <= (1 << 29) && d->M < (1ll << 31) && d->T < (1ll << 31) && d->E <= (1 << 20), "linear: a size beyond what the kernels index");
    const bool x16 = d->x_type == SM_F16 || d->x_type == SM_BF16;
    SM_REQUIRE((x16 && (d->w_type == d->x_type || d->w_type == SM_MX4)) || (d->x_type == SM_MX4 && d->w_type == SM_MX4),
               "linear: x of type %d on weights of type %d (taken: fp16 or bf16 on weights of the same type or MX4, MX4 on MX4)", d->x_type, d->w_type);
    SM_REQUIRE(d->y_type == SM_F32 || ((d->y_type == SM_F16 || d->y_type == SM_BF16) && (!x16 || d->y_type == d->x_type)),
               "linear: output type %d for x of type %d (taken: x's own 16-bit type or fp32; any of the three for an MX4 x)", d->y_type, d->x_type);
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
    p.M = d->M; p.T = d->T; p.N = d->N; p.K = d->T == 0 ? 0 : d->K; p.E = d->E; p.act = d->act; p.slope = d->slope; p.gated = d->gated != 0; p.y_type = d->y_type;
    p.w_rows = p.gated ? 2 * p.N : p.N;
    p.x_ld = x16 && d->x_ld ? 2 * d->x_ld : xr; p.xs_ld = xsr; p.w_ld = wr; p.ws_ld = wsr; p.w_es = wr * p.w_rows; p.ws_es = wsr * p.w_rows; p.y_ld = d->y_ld ? d->y_ld : d->N;
    SM_REQUIRE(d->T <= 1 || p.x_ld >= xr, "linear: row stride of x %lld below its %d columns", (long long)d->x_ld, d->K);
    SM_REQUIRE(d->M == 1 || p.y_ld >= d->N, "linear: row stride of y %lld below its %d columns", p.y_ld, d->N);
    const int ye = d->y_type == SM_F32 ? 4 : 2;
    SM_REQUIRE((size_t)y % ye == 0 && (size_t)bias % 4 == 0 && (size_t)offsets % 4 == 0 && (size_t)rows % 4 == 0 && (!x16 || (size_t)x % 2 == 0) && (d->w_type == SM_MX4 || (size_t)w % 2 == 0),
               "linear: an operand is not aligned to its element");
    SM_REQUIRE((x16 || (size_t)x % 16 == 0) && (d->w_type != SM_MX4 || (size_t)w % 16 == 0), "linear: MX4 codes need 16-byte alignment");
    p.y_vec = (size_t)y % 16 == 0 && p.y_ld * ye % 16 == 0;
    hipStream_t s = sm_s(stream);
    const long long per = p.offsets ? (p.M + p.E - 1) / p.E : p.M;      // rows of an average group
    if (per > 64 && lin_tile_fits(p)) {
        const bool dma = d->x_type == SM_MX4 || (p.K % 8 == 0 && (size_t)x % 16 == 0 && p.x_ld % 16 == 0 && (d->w_type == SM_MX4 || (size_t)w % 16 == 0));
        return lin_tile_launch(p, d->x_type, d->w_type, dma && per > 256 ? 1 : 0, dma, s);
    }
    const int waves = p.K <= 256 ? 1 : p.K <= 1024 ? 4 : 8;
    if (d->x_type == SM_MX4) return lin_stream<SM_MX4, SM_MX4>(p, s, waves);
    if (d->w_type == SM_MX4) return d->x_type == SM_F16 ? lin_stream<SM_F16, SM_MX4>(p, s, waves) : lin_stream<SM_BF16, SM_MX4>(p, s, waves);
    return d->x_type == SM_F16 ? lin_stream<SM_F16, SM_F16>(p, s, waves) : lin_stream<SM_BF16, SM_BF16>(p, s, waves);
}
