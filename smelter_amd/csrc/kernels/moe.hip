// smelter_amd/csrc/kernels/moe.hip — routing of tokens to experts, and the weighted sum of the experts' answers.
//
// Route: per token the k largest of E scores (ties: the lower index first), their softmax weights, and the order of all T k assignments by expert (stable: by token, then by rank), which is what
// the grouped products take:  offsets[e] .. offsets[e + 1] = the slots of expert e,  rows[slot] = token,  slots[token][rank] = slot.  A score of -inf or NaN is never chosen: a token with fewer
// than k others gets expert -1, weight 0 and slot -1 for the rest, a padded token (all -inf) no slot at all.  Weights: exp(z_i - z_max) over the sum of the chosen ones (renormalised) or of all
// E; a score that equals the maximum counts as 1, so +inf scores share the weight.  Statistics in fp32.
//
// The order is a counting sort in which every place is computed, none handed out by an atomic's order.  Up to SMALL assignments one block does everything in one launch; above, one launch selects
// and counts per block, a second adds the counts of the blocks before it and places.  Bound by latency: 8 of 128 bf16 scores for 16384 tokens take 10.5 us (k dependent rounds of a maximum over 16
// lanes) and 8.4 us, 6 of 64 fp32 scores for 7 tokens 5.7 us.
#include "linear.hpp"

#define MOE_MAX_E 1024
#define MOE_MAX_K 32

struct RouteParams {
    const char* z; int type; long long T; int E, k; long long ld; int renorm;       // ld in elements
    float* weights; int* experts; int* offsets; int* rows; int* slots; int* counts;
    int per_block;                                                                    // tokens of a block
};

// scores as unsigned keys in their order; 0 = never chosen
__device__ __forceinline__ unsigned route_key(float z) {
    if (!(z > -__builtin_inff())) return 0;
    const unsigned b = __builtin_bit_cast(unsigned, z);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float route_value(unsigned key) { return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ float route_load(const RouteParams& p, long long t, int e) {
    const long long i = t * p.ld + e;
    return p.type == SM_F32 ? ((const float*)p.z)[i] : p.type == SM_F16 ? (float)((const half_t*)p.z)[i] : (float)((const bf16_t*)p.z)[i];
}

// maximum / minimum / sum over the 16 lanes of a row, in every one of them (rotations inside the row: no LDS)
template <class F> __device__ __forceinline__ unsigned route_row(unsigned v, F f) {
    v = f(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true)); v = f(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));
    v = f(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true)); return f(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));
}
__device__ __forceinline__ unsigned route_max(unsigned v) { return route_row(v, [](unsigned a, unsigned b) { return a > b ? a : b; }); }
__device__ __forceinline__ unsigned route_min(unsigned v) { return route_row(v, [](unsigned a, unsigned b) { return a < b ? a : b; }); }
__device__ __forceinline__ float route_sum(float v) {
    return __builtin_bit_cast(float, route_row(__builtin_bit_cast(unsigned, v), [](unsigned a, unsigned b) { return __builtin_bit_cast(unsigned, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b)); }));
}

// Four tokens by one wave, each by a row of 16 lanes: lane l of a row holds the scores of experts l, 16 + l, ...  (one token by a whole wave with shuffles: 64 us for 16384 tokens of 128 scores.)
// t >= t1: no token (its lanes run along).
template <int EPL> __device__ __forceinline__ void route_tokens(const RouteParams& p, long long t, long long t1, int* hist) {
    const int l = threadIdx.x & 15;
    const bool in = t < t1;
    unsigned key[EPL];
#pragma unroll
    for (int j = 0; j < EPL; j++) { const int e = j * 16 + l; float z = in && e < p.E ? route_load(p, t, e) : -__builtin_inff(); if (z == 0.f) z = 0.f; key[j] = route_key(z); }
    unsigned first = 0; float total = 0.f;
    if (!p.renorm) {                                                               // the maximum first: the sum goes over all scores
#pragma unroll
        for (int j = 0; j < EPL; j++) first = first > key[j] ? first : key[j];
        first = route_max(first);
#pragma unroll
        for (int j = 0; j < EPL; j++) total += key[j] == 0 ? 0.f : key[j] == first ? 1.f : expf(route_value(key[j]) - route_value(first));
        total = route_sum(total);
    }
    float mine[2] = {0.f, 0.f}; int expert[2] = {-1, -1};                           // lane l keeps the choices l and 16 + l
    for (int i = 0; i < p.k; i++) {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < EPL; j++) m = m > key[j] ? m : key[j];
        m = route_max(m);
        if (i == 0) first = m;
        unsigned at = ~0u;                                                          // the lowest expert with that score
#pragma unroll
        for (int j = EPL - 1; j >= 0; j--) at = key[j] == m ? (unsigned)(j * 16 + l) : at;
        at = route_min(at);
#pragma unroll
        for (int j = 0; j < EPL; j++) key[j] = (unsigned)(j * 16 + l) == at ? 0 : key[j];
        const float e1 = m == 0 ? 0.f : m == first ? 1.f : expf(route_value(m) - route_value(first));
        if (p.renorm) total += e1;
        if ((i & 15) == l) { if (i < 16) { mine[0] = e1; expert[0] = m == 0 ? -1 : (int)at; } else { mine[1] = e1; expert[1] = m == 0 ? -1 : (int)at; } }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int i = 16 * h + l;
        if (!in || i >= p.k) continue;
        p.experts[t * p.k + i] = expert[h];
        p.weights[t * p.k + i] = expert[h] < 0 ? 0.f : mine[h] / total;
        if (expert[h] >= 0) atomicAdd(&hist[expert[h]], 1);                         // a count: the same in any order
    }
}

// Places the assignments a0 .. a1 of this block: `start[e]` = slot of the first one of expert e.  Each wave takes a run of them in order; waves before it are counted first.
__device__ __forceinline__ void route_place(const RouteParams& p, const int* experts, long long a0, int n, int* start, int* wcount) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int per = ((n + waves - 1) / waves + 63) & ~63;
    const int lo = wave * per < n ? wave * per : n, hi = lo + per < n ? lo + per : n;
    for (int i = threadIdx.x; i < waves * p.E; i += blockDim.x) wcount[i] = 0;
    __syncthreads();
    for (int i = lo + lane; i < hi; i += 64) { const int e = experts[a0 + i]; if (e >= 0) atomicAdd(&wcount[wave * p.E + e], 1); }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) { int s = start[e]; for (int w = 0; w < waves; w++) { const int c = wcount[w * p.E + e]; wcount[w * p.E + e] = s; s += c; } }
    __syncthreads();
    const int bits = 32 - __builtin_clz(p.E);
    for (int i0 = lo; i0 < hi; i0 += 64) {
        const int i = i0 + lane;
        const int e = i < hi ? experts[a0 + i] : -1;
        unsigned long long same = __ballot(e >= 0);
        if (e < 0) same = 0;
        for (int b = 0; b < bits; b++) { const unsigned long long v = __ballot(e >= 0 && (e >> b & 1)); same &= (e >> b & 1) ? v : ~v; }
        const int before = __popcll(same & ((1ull << lane) - 1));
        int slot = -1;
        if (e >= 0) slot = wcount[wave * p.E + e] + before;
        __builtin_amdgcn_wave_barrier();
        if (e >= 0 && (same >> lane) == 1ull) wcount[wave * p.E + e] = slot + 1;       // the last lane of its expert
        __builtin_amdgcn_wave_barrier();
        if (i < hi) { p.slots[a0 + i] = slot; if (e >= 0) p.rows[slot] = (int)((a0 + i) / p.k); }
    }
}

// exclusive prefix sum of total[0 .. E) into offs[0 .. E] by the first wave of the block
__device__ __forceinline__ void route_scan(const int* total, int* offs, int E) {
    if (threadIdx.x >= 64) return;
    int run = 0;
    for (int base = 0; base < E; base += 64) {
        const int e = base + threadIdx.x, v = e < E ? total[e] : 0;
        int s = v;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int up = __shfl_up(s, d); if ((int)threadIdx.x >= d) s += up; }
        if (e < E) offs[e] = run + s - v;
        run += __shfl(s, 63);
    }
    if (threadIdx.x == 0) offs[E] = run;
}

// ONE = true: the whole of a small routing in one block
template <int EPL, bool ONE> __global__ __launch_bounds__(EPL <= 16 ? 1024 : 512) void route_select_kernel(RouteParams p) {
    extern __shared__ int lds[];
    int* hist = lds;                                                             // [E]
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    const long long t0 = (long long)blockIdx.x * p.per_block, t1 = t0 + p.per_block < p.T ? t0 + p.per_block : p.T;
    for (long long t = t0 + wave * 4; t < t1; t += waves * 4) route_tokens<EPL>(p, t + ((threadIdx.x & 63) >> 4), t1, hist);
    __syncthreads();
    if constexpr (!ONE) { for (int e = threadIdx.x; e < p.E; e += blockDim.x) p.counts[(long long)blockIdx.x * p.E + e] = hist[e]; }
    else {
        int* offs = lds + p.E; int* wcount = offs + p.E + 1;
        route_scan(hist, offs, p.E);
        __threadfence_block();
        __syncthreads();
        for (int e = threadIdx.x; e <= p.E; e += blockDim.x) p.offsets[e] = offs[e];
        const int used = offs[p.E], n = (int)(p.T * p.k);
        for (int i = used + threadIdx.x; i < n; i += blockDim.x) p.rows[i] = -1;
        route_place(p, p.experts, 0, n, offs, wcount);
    }
}

__global__ __launch_bounds__(1024) void route_place_kernel(RouteParams p, int blocks) {
    extern __shared__ int lds[];
    int* total = lds; int* before = total + p.E; int* offs = before + p.E; int* wcount = offs + p.E + 1;
    for (int e = threadIdx.x; e < 2 * p.E; e += blockDim.x) lds[e] = 0;
    __syncthreads();
    // counts of all blocks and of the blocks before this one (integer sums, the same in any order): a thread adds one expert's over every parts-th block, sixteen loads at a time
    const int parts = (int)blockDim.x / p.E > 0 ? (int)blockDim.x / p.E : 1;
    for (int i = threadIdx.x; i < parts * p.E; i += blockDim.x) {
        const int e = i % p.E, part = i / p.E;
        int all = 0, low = 0;
        for (int b0 = part; b0 < blocks; b0 += 16 * parts) {
            int c[16];
#pragma unroll
            for (int q = 0; q < 16; q++) { const int b = b0 + q * parts; c[q] = b < blocks ? p.counts[(long long)b * p.E + e] : 0; }
#pragma unroll
            for (int q = 0; q < 16; q++) { all += c[q]; low += b0 + q * parts < (int)blockIdx.x ? c[q] : 0; }
        }
        if (all) atomicAdd(&total[e], all);
        if (low) atomicAdd(&before[e], low);
    }
    __syncthreads();
    route_scan(total, offs, p.E);
    __syncthreads();
    const int used = offs[p.E];
    if (blockIdx.x == 0) for (int e = threadIdx.x; e <= p.E; e += blockDim.x) p.offsets[e] = offs[e];
    for (long long i = used + (long long)blockIdx.x * blockDim.x + threadIdx.x; i < p.T * p.k; i += (long long)gridDim.x * blockDim.x) p.rows[i] = -1;
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) before[e] += offs[e];
    __syncthreads();
    const long long t0 = (long long)blockIdx.x * p.per_block, t1 = t0 + p.per_block < p.T ? t0 + p.per_block : p.T;
    route_place(p, p.experts, t0 * p.k, (int)((t1 - t0) * p.k), before, wcount);
}

#define ROUTE_SMALL 64                                                            // tokens

static long long route_blocks(long long T, int* per) {
    long long b = (T + 63) / 64; if (b > 512) b = 512;
    *per = (int)((T + b - 1) / b);
    return (T + *per - 1) / *per;
}

extern "C" size_t sm_moe_route_workspace_bytes(int64_t T, int32_t E, int32_t k) {
    if (T <= ROUTE_SMALL || E < 1) return 0;
    int per; return (size_t)route_blocks(T, &per) * E * sizeof(int);
}

template <int EPL> static int route_launch(RouteParams p, hipStream_t s) {
    constexpr int WAVES = EPL <= 16 ? 16 : 8;                                     // of the selecting kernel: 64 tokens at once, 32 where a lane holds more scores
    if (p.T <= ROUTE_SMALL) {
        p.per_block = (int)p.T;
        route_select_kernel<EPL, true><<<1, 64 * WAVES, p.E * sizeof(int) + (size_t)(WAVES * p.E + p.E + 1) * sizeof(int), s>>>(p);
    } else {
        const long long blocks = route_blocks(p.T, &p.per_block);
        route_select_kernel<EPL, false><<<dim3((unsigned)blocks), 64 * WAVES, p.E * sizeof(int), s>>>(p);
        SM_LAUNCH_CHECK();
        // waves of the placing one: more to add the counts of many blocks (16384 tokens of 256 scores: 26.4 us with 16, 30.6 with 8), fewer to count and join (1024 of 128: 15.1, 13.9); 8 is what
        // LDS holds of more than 256 experts
        const int place = EPL <= 16 && blocks >= 128 ? 16 : 8;
        route_place_kernel<<<dim3((unsigned)blocks), 64 * place, (size_t)((place + 3) * p.E + 1) * sizeof(int), s>>>(p, (int)blocks);
    }
    SM_LAUNCH_CHECK();
    return SM_OK;
}

extern "C" int sm_moe_route(const void* scores, int32_t type, int64_t T, int32_t E, int32_t k, int64_t ld, int32_t renormalize, float* weights, int32_t* experts, int32_t* offsets,
                            int32_t* rows, int32_t* slots, void* workspace, size_t workspace_bytes, sm_stream_t stream) {
    SM_REQUIRE(type == SM_F16 || type == SM_BF16 || type == SM_F32, "moe_route: type %d is not fp16, bf16 or fp32", type);
    SM_REQUIRE(E >= 1 && E <= MOE_MAX_E, "moe_route: %d experts (taken: 1 .. %d)", E, MOE_MAX_E);
    SM_REQUIRE(k >= 1 && k <= MOE_MAX_K && k <= E, "moe_route: %d of %d experts (taken: 1 .. min(%d, E))", k, E, MOE_MAX_K);
    SM_REQUIRE(T >= 0 && T < (1ll << 31) && T * k < (1ll << 31), "moe_route: %lld tokens x %d", (long long)T, k);
    SM_REQUIRE(offsets && (T == 0 || (scores && weights && experts && rows && slots)), "moe_route: null operand");
    SM_REQUIRE(T <= 1 || ld >= E, "moe_route: row stride %lld below the %d scores", (long long)ld, E);
    SM_REQUIRE((size_t)scores % (type == SM_F32 ? 4 : 2) == 0, "moe_route: scores are not aligned to their element");
    SM_REQUIRE(workspace_bytes >= sm_moe_route_workspace_bytes(T, E, k) && (workspace || T <= ROUTE_SMALL) && (size_t)workspace % 4 == 0, "moe_route: workspace of %zu bytes, %zu wanted",
               workspace_bytes, sm_moe_route_workspace_bytes(T, E, k));
    RouteParams p = {};
    p.z = (const char*)scores; p.type = type; p.T = T; p.E = E; p.k = k; p.ld = ld; p.renorm = renormalize;
    p.weights = weights; p.experts = experts; p.offsets = offsets; p.rows = rows; p.slots = slots; p.counts = (int*)workspace;
    hipStream_t s = sm_s(stream);
    if (E <= 64) return route_launch<4>(p, s);
    if (E <= 128) return route_launch<8>(p, s);
    if (E <= 256) return route_launch<16>(p, s);
    if (E <= 512) return route_launch<32>(p, s);
    return route_launch<64>(p, s);
}

// out[t, n] = sum_j weights[t, j] * y[slots[t, j], n]: one thread per eight columns of a token, terms added in the order of j in fp32, one rounding; a slot outside 0 .. M - 1 adds nothing.
// Bound by the reading of the k rows: 16384 x 8 rows of 2048 in bf16 take 122 us (4.9 TB/s).
template <int KIND> __device__ __forceinline__ void combine_load8(const char* row, int c, int N, float* v) {
    if constexpr (KIND == SM_F32) {
        const float* q = (const float*)row + c;
        if (c + 8 <= N) __builtin_memcpy(v, q, 32);
        else for (int i = 0; i < 8; i++) v[i] = c + i < N ? q[i] : 0.f;
    } else {
        const intx4_t b = lin_load8(row, c, N);
        if constexpr (KIND == SM_F16) { const half8_t h = __builtin_bit_cast(half8_t, b); for (int i = 0; i < 8; i++) v[i] = (float)h[i]; }
        else { const bf16x8_t h = __builtin_bit_cast(bf16x8_t, b); for (int i = 0; i < 8; i++) v[i] = (float)h[i]; }
    }
}
template <int KIND> __global__ void combine_kernel(const char* y, long long M, int N, long long y_ld, const float* weights, const int* slots, long long T, int k, void* out, int out_type, long long out_ld,
                                                   int vec) {
    const int chunks = (N + 7) / 8;
    const long long units = T * chunks;
    for (long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x; u < units; u += (long long)gridDim.x * blockDim.x) {
        const long long t = u < 0x7fffffffll ? (long long)((unsigned)u / (unsigned)chunks) : u / chunks;
        const int c = (int)(u - t * chunks) * 8;
        float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int j = 0; j < k; j++) {
            const int at = slots[t * k + j];
            if (at < 0 || at >= M) continue;
            const float w = weights[t * k + j];
            float v[8]; combine_load8<KIND>(y + (KIND == SM_F32 ? 4ll : 2ll) * at * y_ld, c, N, v);
            for (int i = 0; i < 8; i++) s[i] += w * v[i];
        }
        const long long o = t * out_ld + c;
        if (vec && c + 8 <= N) lin_store8(out, o, s, out_type);
        else for (int i = 0; i < 8; i++) if (c + i < N) lin_store1(out, o + i, s[i], out_type);
    }
}

extern "C" int sm_moe_combine(const void* y, int32_t type, int64_t M, int32_t N, int64_t y_ld, const float* weights, const int32_t* slots, int64_t T, int32_t k, void* out, int32_t out_type,
                              int64_t out_ld, sm_stream_t stream) {
    SM_REQUIRE((type == SM_F16 || type == SM_BF16 || type == SM_F32) && (out_type == SM_F16 || out_type == SM_BF16 || out_type == SM_F32), "moe_combine: types %d -> %d (taken: fp16, bf16, fp32)", type, out_type);
    SM_REQUIRE(M >= 0 && N >= 0 && T >= 0 && k >= 0 && M < (1ll << 31) && T < (1ll << 31) && N <= (1 << 29), "moe_combine: sizes M %lld, N %d, T %lld, k %d", (long long)M, N, (long long)T, k);
    if (T == 0 || N == 0) return SM_OK;
    SM_REQUIRE(out && (k == 0 || (weights && slots)) && (k == 0 || M == 0 || y), "moe_combine: null operand");
    SM_REQUIRE((M <= 1 || y_ld >= N) && (T == 1 || out_ld >= N), "moe_combine: row strides %lld, %lld below the %d columns", (long long)y_ld, (long long)out_ld, N);
    const int oe = out_type == SM_F32 ? 4 : 2;
    SM_REQUIRE((size_t)y % (type == SM_F32 ? 4 : 2) == 0 && (size_t)out % oe == 0, "moe_combine: an operand is not aligned to its element");
    const int vec = (size_t)out % 16 == 0 && (T == 1 || out_ld * oe % 16 == 0);
    const long long units = T * ((N + 7) / 8), want = (units + 255) / 256, cap = (long long)SM_NUM_CU * 32;
    const dim3 grid((unsigned)(want < cap ? want : cap));
    if (type == SM_F16) combine_kernel<SM_F16><<<grid, 256, 0, sm_s(stream)>>>((const char*)y, M, N, y_ld, weights, slots, T, k, out, out_type, out_ld, vec);
    else if (type == SM_BF16) combine_kernel<SM_BF16><<<grid, 256, 0, sm_s(stream)>>>((const char*)y, M, N, y_ld, weights, slots, T, k, out, out_type, out_ld, vec);
    else combine_kernel<SM_F32><<<grid, 256, 0, sm_s(stream)>>>((const char*)y, M, N, y_ld, weights, slots, T, k, out, out_type, out_ld, vec);
    SM_LAUNCH_CHECK();
    return SM_OK;
}
