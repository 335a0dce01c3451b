// The router of a mixture of experts: logits = x W^T, the top_k experts of every row and their weights.  The choice compares values that
// can lie closer than fp32 sums are exact, so the logits are summed in 64 bits and rounded once; equal ones go to the lowest
// index.
#include "step_dev.h"
#include "step_mix_launch.h"

#include <algorithm>

namespace qkv {
namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int RW = 8; // waves of a workgroup of k_route_logits

// A workgroup per (16 experts, 16 rows, chunk of dim): its waves take every RW-th step of 32 values, by matrix instructions in 64 bits
// (lane n = lane & 15 holds 8 values of expert and row n from 8 (lane / 16) on; one instruction for each of the 8), and add up in LDS.
template <int DT, int WT> __global__ __launch_bounds__(RW * 64) void k_route_logits(RouteArgs a) {
    __shared__ double red[RW * 256];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int e0 = blockIdx.x * 16, row0 = blockIdx.y * 16, steps = (a.dim + 31) >> 5;
    const int s0 = (int) ((long long) steps * blockIdx.z / a.chunks), s1 = (int) ((long long) steps * (blockIdx.z + 1) / a.chunks);
    const typename Elem<WT>::T * wp = static_cast<const typename Elem<WT>::T *>(a.w) + (size_t) min(e0 + n, a.n_experts - 1) * a.dim;
    const typename Elem<DT>::T * xp = static_cast<const typename Elem<DT>::T *>(a.x) + min(row0 + n, a.rows - 1) * a.x_stride;
    f64x4 acc = {0, 0, 0, 0};
    for (int s = s0 + wave; s < s1; s += RW) {
        const int k = 32 * s + 8 * g;
        float w[8], x[8];
        if (k + 8 <= a.dim) {
            load8<WT>(wp + k, w);
            load8<DT>(xp + k, x);
        } else {
            load_n<WT>(wp + k, max(a.dim - k, 0), w);
            load_n<DT>(xp + k, max(a.dim - k, 0), x);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double) w[i], (double) x[i], acc, 0, 0, 0);
    }
    // lane n: row n, register r: expert g + 4 r
#pragma unroll
    for (int r = 0; r < 4; r++) red[wave * 256 + n * 16 + g + 4 * r] = acc[r];
    __syncthreads();
    if (threadIdx.x >= 256) return;
    double v = 0;
#pragma unroll
    for (int w = 0; w < RW; w++) v += red[w * 256 + threadIdx.x];
    const int row = row0 + (threadIdx.x >> 4), e = e0 + (threadIdx.x & 15);
    if (row >= a.rows || e >= a.n_experts) return;
    const size_t at = (size_t) row * a.n_experts + e;
    if (a.chunks > 1) a.part[(size_t) blockIdx.z * a.rows * a.n_experts + at] = v;
    else a.logits[at] = (float) v;
}

// a double's order as an unsigned one; NaN below everything
__device__ __forceinline__ uint64_t order(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v == 0 ? 0.0 : v);
    return v != v ? 0 : b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ uint64_t shfl_xor_64(uint64_t v, int m) {
    return (uint64_t) shfl_xor_u((unsigned) (v >> 32), m) << 32 | shfl_xor_u((unsigned) v, m);
}

constexpr int PW = 4; // rows (waves) of a workgroup of k_route_pick

// A wave per row, lane l holds experts l, l + 64, ...: V a lane.
template <int V> __global__ __launch_bounds__(PW * 64) void k_route_pick(RouteArgs a) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int row = blockIdx.x * PW + wave;
    if (row >= a.rows) return;
    float l[V];
    double score[V];
    uint64_t key[V];
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = lane + 64 * i;
        const size_t at = (size_t) row * a.n_experts + e;
        l[i] = -__builtin_inff();
        score[i] = 0;
        key[i] = 0;
        if (e >= a.n_experts) continue;
        if (a.chunks > 1) {
            double v = 0;
            for (int c = 0; c < a.chunks; c++) v += a.part[(size_t) c * a.rows * a.n_experts + at];
            a.logits[at] = l[i] = (float) v;
        } else l[i] = a.logits[at];
        score[i] = l[i];
        if (a.form >= ROUTE_SIGMOID) score[i] = 1.0 / (1.0 + exp(-(double) l[i]));
        key[i] = order(a.bias ? score[i] + (double) a.bias[e] : (double) l[i]);
        top = fmaxf(top, l[i]);
    }
    // the largest key, the lowest index of equal ones, top_k times; lane j keeps the j-th
    unsigned taken = 0;
    int mine_id = 0;
    double mine = 0;
    for (int j = 0; j < a.top_k; j++) {
        uint64_t best = 0;
        int at = 0x7fffffff;
        double s = 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int e = lane + 64 * i;
            if (e < a.n_experts && !(taken >> i & 1) && (at == 0x7fffffff || key[i] > best)) best = key[i], at = e, s = score[i];
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint64_t k = shfl_xor_64(best, m);
            const int e = (int) shfl_xor_u((unsigned) at, m);
            const double t = shfl_xor_d(s, m);
            if (k > best || (k == best && e < at)) best = k, at = e, s = t;
        }
        if ((at & 63) == lane) taken |= 1u << (at >> 6);
        if (lane == j) mine_id = at, mine = s;
    }
    const bool in = lane < a.top_k;
    double w = mine;
    if (a.form == ROUTE_SOFTMAX) {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, shfl_xor(top, m));
        double sum = 0;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (lane + 64 * i < a.n_experts) sum += exp((double) l[i] - (double) top);
        w = exp(mine - (double) top) / wave_sum(sum);
    } else if (a.form == ROUTE_CHOSEN) {
        // (the first one is the largest)
        const uint64_t b = __builtin_bit_cast(uint64_t, mine);
        const double first = __builtin_bit_cast(double, (uint64_t) (unsigned) __builtin_amdgcn_readfirstlane((unsigned) (b >> 32)) << 32 |
                                                            (unsigned) __builtin_amdgcn_readfirstlane((unsigned) b));
        const double e = in ? exp(mine - first) : 0.0;
        w = e / wave_sum(e);
    } else if (a.form == ROUTE_SIGMOID_NORM) w = mine / wave_sum(in ? mine : 0.0);
    if (in) {
        a.ids[(size_t) row * a.top_k + lane] = mine_id;
        a.weights[(size_t) row * a.top_k + lane] = (float) (w * (double) a.scale);
    }
}

template <int DT, int WT> hipError_t logits(const RouteArgs & a, hipStream_t st) {
    return launch(k_route_logits<DT, WT>, dim3((a.n_experts + 15) / 16, (a.rows + 15) / 16, a.chunks), dim3(RW * 64), 0, st, a);
}
template <int DT> hipError_t logits(const RouteArgs & a, int wtype, hipStream_t st) {
    return wtype == DT_F32 ? logits<DT, DT_F32>(a, st) : wtype == DT_F16 ? logits<DT, DT_F16>(a, st) : logits<DT, DT_BF16>(a, st);
}

} // namespace

void route_plan(RouteArgs & a) { a.chunks = 1; }

hipError_t launch_route(const RouteArgs & a, int dtype, int wtype, hipStream_t st) {
    const hipError_t e = dtype == DT_F32 ? logits<DT_F32>(a, wtype, st) : dtype == DT_F16 ? logits<DT_F16>(a, wtype, st) : logits<DT_BF16>(a, wtype, st);
    if (e != hipSuccess) return e;
    const dim3 grid((a.rows + PW - 1) / PW), block(PW * 64);
    const int v = (a.n_experts + 63) / 64;
    return v <= 1 ? launch(k_route_pick<1>, grid, block, 0, st, a) : v <= 2 ? launch(k_route_pick<2>, grid, block, 0, st, a)
         : v <= 4 ? launch(k_route_pick<4>, grid, block, 0, st, a) : launch(k_route_pick<16>, grid, block, 0, st, a);
}

} // namespace qkv
