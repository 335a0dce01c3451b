// The router of a mixture of experts: logits = x W^T, the top_k experts of every row and their weights.  The choice compares values that
// can lie closer than fp32 sums are exact, so the logits are summed in 64 bits and rounded once; equal ones go to the lowest
// index.
#include "step_route_dev.h"

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

constexpr int PW = 4; // rows (waves) of a workgroup of k_route_pick

template <int V> __global__ __launch_bounds__(PW * 64) void k_route_pick(RouteArgs a) {
    const int row = blockIdx.x * PW + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row < a.rows) route_pick<V>(a, row);
}

template <int DT, int WT> hipError_t logits(const RouteArgs & a, hipStream_t st) {
    return launch(k_route_logits<DT, WT>, dim3((a.n_experts + 15) / 16, (a.rows + 15) / 16, a.chunks), dim3(RW * 64), 0, st, a);
}
template <int DT> hipError_t logits(const RouteArgs & a, int wtype, hipStream_t st) {
    return wtype == DT_F32 ? logits<DT, DT_F32>(a, st) : wtype == DT_F16 ? logits<DT, DT_F16>(a, st) : logits<DT, DT_BF16>(a, st);
}

} // namespace

void route_plan(RouteArgs & a) {
    // few tiles: dim in chunks of at least a step a wave, up to two workgroups a CU (and 16 KiB of partial sums an expert)
    const int tiles = ((a.n_experts + 15) / 16) * ((a.rows + 15) / 16), steps = (a.dim + 31) / 32;
    a.chunks = std::max(1, std::min({ROUTE_MAX_CHUNKS, 512 / std::max(tiles, 1), steps / RW, 2048 / std::max(a.rows, 1)}));
}

hipError_t launch_logits(const RouteArgs & a, int dtype, int wtype, hipStream_t st) {
    return dtype == DT_F32 ? logits<DT_F32>(a, wtype, st) : dtype == DT_F16 ? logits<DT_F16>(a, wtype, st) : logits<DT_BF16>(a, wtype, st);
}
hipError_t launch_pick(const RouteArgs & a, hipStream_t st) {
    const dim3 grid((a.rows + PW - 1) / PW), block(PW * 64);
    const int v = (a.n_experts + 63) / 64;
    return v <= 1 ? launch(k_route_pick<1>, grid, block, 0, st, a) : v <= 2 ? launch(k_route_pick<2>, grid, block, 0, st, a)
         : v <= 4 ? launch(k_route_pick<4>, grid, block, 0, st, a) : launch(k_route_pick<16>, grid, block, 0, st, a);
}

} // namespace qkv
