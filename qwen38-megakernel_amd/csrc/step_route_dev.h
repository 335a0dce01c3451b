// The choice of a row's experts from its logits, by one wave (k_route_pick, and the experts' k_moe_prep).
#pragma once
#include "step_dev.h"
#include "step_mix_launch.h"

namespace qkv {

// the largest value of the wave's lanes: rows of 16 lanes, then rows 0 and 1, 2 and 3, then both halves, in lane 63
__device__ __forceinline__ unsigned wave_max_u(unsigned v) {
    v = max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x111, 0xf, 0xf, true)); // row_shr:1
    v = max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x112, 0xf, 0xf, true)); // row_shr:2
    v = max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x114, 0xf, 0xf, true)); // row_shr:4
    v = max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x118, 0xf, 0xf, true)); // row_shr:8
    v = max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x142, 0xa, 0xf, true)); // row_bcast:15
    v = max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x143, 0xc, 0xf, true)); // row_bcast:31
    return (unsigned) __builtin_amdgcn_readlane((int) v, 63);
}
// the order of floats as unsigned ones; a NaN below everything, and everything above 0
__device__ __forceinline__ unsigned order32(float v) {
    const unsigned b = __builtin_bit_cast(unsigned, v == 0.f ? 0.f : v);
    return v != v ? 1 : b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v == 0 ? 0.0 : v);
    return v != v ? 1 : b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double sigmoid_d(double v) { return 1.0 / (1.0 + exp(-v)); }

// the choice of one row from its logits in registers, lane l holding experts V l .. V l + V - 1 (of equal keys the lowest index is then the lowest
// lane's first): lane j keeps the j-th, up to `most` of them
template <int V> struct Chosen {
    int expert;
    float logit;
};
template <int V> __device__ __forceinline__ Chosen<V> route_choose(const RouteArgs & a, const float (&l)[V], int most) {
    const int lane = threadIdx.x & 63;
    unsigned hi[V], lo[V]; // keys, 0 for no expert and for those taken; without a bias the logits' order alone
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = lane * V + i;
        if (a.bias) {
            const uint64_t k = order64(sigmoid_d(l[i]) + (double) a.bias[min(e, a.n_experts - 1)]);
            hi[i] = (unsigned) (k >> 32);
            lo[i] = (unsigned) k;
        } else hi[i] = order32(l[i]), lo[i] = 0;
        if (e >= a.n_experts) hi[i] = lo[i] = 0;
    }
    Chosen<V> c{0, 0.f};
    for (int j = 0; j < most; j++) {
        unsigned h = hi[0], w = lo[0];
        int at = 0;
        float v = l[0];
#pragma unroll
        for (int i = 1; i < V; i++)
            if (hi[i] > h || (hi[i] == h && lo[i] > w)) h = hi[i], w = lo[i], at = i, v = l[i];
        uint64_t best = __ballot(h == wave_max_u(h));
        if (a.bias && (best & (best - 1))) { // (more lanes than one with the upper half)
            const bool in = best >> lane & 1;
            const unsigned m = wave_max_u(in ? w : 0);
            best = __ballot(in && w == m);
        }
        const int who = __builtin_ctzll(best), e = who * V + __builtin_amdgcn_readlane(at, who);
        const float ve = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), who));
#pragma unroll
        for (int i = 0; i < V; i++)
            if (e == lane * V + i) hi[i] = lo[i] = 0;
        if (lane == j) c.expert = e, c.logit = ve;
    }
    return c;
}
// its weights, and both to memory
template <int V> __device__ __forceinline__ void route_weights(const RouteArgs & a, int row, const float (&l)[V], const Chosen<V> & c) {
    const int lane = threadIdx.x & 63;
    const bool in = lane < a.top_k;
    double w;
    if (a.form == ROUTE_SOFTMAX) {
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < V; i++)
            if (lane * V + i < a.n_experts) top = fmaxf(top, l[i]);
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, shfl_xor(top, m));
        double sum = 0;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (lane * V + i < a.n_experts) sum += exp((double) l[i] - (double) top);
        w = exp((double) c.logit - (double) top) / wave_sum(sum);
    } else if (a.form == ROUTE_CHOSEN) {
        const float top = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, c.logit))); // (the first is the largest)
        const double e = in ? exp((double) c.logit - (double) top) : 0.0;
        w = e / wave_sum(e);
    } else {
        // (where all the chosen ones lie far below zero sigmoids are exponentials to 64 bits, and may leave their range: relative to the largest)
        const bool far = a.form == ROUTE_SIGMOID_NORM && !__any(in && c.logit >= -600.f);
        float top = in ? c.logit : -__builtin_inff();
        if (far)
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, shfl_xor(top, m));
        w = !in ? 0.0 : far ? exp((double) c.logit - (double) top) : sigmoid_d(c.logit);
        if (a.form == ROUTE_SIGMOID_NORM) w /= wave_sum(w);
    }
    if (in) {
        a.ids[(size_t) row * a.top_k + lane] = c.expert;
        a.weights[(size_t) row * a.top_k + lane] = (float) (w * (double) a.scale);
    }
}

// Row `row`'s top_k experts and their weights from the logits, or their partial sums; lane j returns the j-th expert (j < top_k).
template <int V> __device__ __forceinline__ int route_pick(const RouteArgs & a, int row) {
    const int lane = threadIdx.x & 63;
    const size_t r0 = (size_t) row * a.n_experts;
    float l[V];
    if (a.chunks > 1) {
        double s[V];
#pragma unroll
        for (int i = 0; i < V; i++) s[i] = 0;
#pragma unroll 4
        for (int c = 0; c < a.chunks; c++)
#pragma unroll
            for (int i = 0; i < V; i++) s[i] += a.part[(size_t) c * a.rows * a.n_experts + r0 + min(lane * V + i, a.n_experts - 1)];
#pragma unroll
        for (int i = 0; i < V; i++) {
            l[i] = (float) s[i];
            if (lane * V + i < a.n_experts) a.logits[r0 + lane * V + i] = l[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) l[i] = a.logits[r0 + min(lane * V + i, a.n_experts - 1)];
    }
    const Chosen<V> c = route_choose<V>(a, l, a.top_k);
    route_weights<V>(a, row, l, c);
    return c.expert;
}

} // namespace qkv
