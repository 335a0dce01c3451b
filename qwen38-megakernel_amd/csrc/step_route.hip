// The router of a mixture of experts: logits = x W^T, the top_k experts of every row and their weights.  The choice compares values that
// can lie closer than fp32 sums are exact, so the logits are summed in 64 bits and rounded once; equal ones go to the lowest
// index.  Many rows of 16-bit types take a shorter way to the same choice (k_route_many): sums in fp32, with a bound on their error, and 64 bits
// for those that lie closer to another than the bound can tell apart.
//
// One bf16 row, 128 experts of 5,120: 8.4 us, two launches' chains.  64 fp32 rows, 256 experts with a bias: 18 us, half of it the choice (a wave a row;
// matrix instructions in 64 bits 30% busy).  4,096 bf16 rows, 63 experts of 2,048: 18 us.
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

// Many rows: a workgroup has 16 rows and all experts, 256 values of dim at a time in LDS, copied 32 lanes a row (an operand's 64 lanes are 16 rows;
// loaded from memory as such, a cache line each, 4,096 rows of 2,048 x 63 experts take 21.0 us, so 17.9).  Its 16 waves take tiles of 16 experts
// (few tiles: parts of dim), sums in fp32 by 16-bit matrix instructions, whose products are exact; two more give the squares of the rows' and the
// experts' norms.  An instruction rounds its products' sum, which |x| |w| bounds, and the sum so far: a chain of c of them is off by less than
// (c + 40) 2^-22 |x| |w|.  Experts of a row that are among the first top_k, or within twice that of them, and lie that close to another of those,
// are summed again in 64 bits by all waves together; the others' order is certain.
constexpr int MW = 16; // waves of a workgroup, one for a row's choice
// Rows from which it is taken.  A workgroup a CU up to 4,096 rows, its time hardly grows with them (bf16, us; behind it k_route_logits and k_route_pick):
// 63 x 2,048: 1,024 rows 17.0, 13.5; 1,536 17.7, 19.0; 4,096 18.0, 29.  128 x 5,120: 41, 37; 44, 50; 44, 111.  256 x 7,168: 109, 84; 111, 118.  Small ones
// gain later (8 x 2,048, 1,536 rows: 14.9, 12.2; 256 x 512 21.7, 19.0, and of 2,048 rows 21.7, 21.9).
constexpr int MANY_ROWS = 1536;
template <int DT> __device__ __forceinline__ f32x4 mfma16(const typename Elem<DT>::Raw8 & a, const typename Elem<DT>::Raw8 & b, f32x4 c) {
    if constexpr (DT == DT_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else {
        typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
}
template <int V> struct Sums { // of 16 rows, in the place of the values
    float part[MW * 256], logit[16 * V * 64], xsq[MW][16], wsq[MW][V * 64];
    uint16_t list[16 * V * 64];
    int count;
};
template <int DT, int V> __global__ __launch_bounds__(MW * 64) void k_route_many(RouteArgs a) {
    typedef typename Elem<DT>::T T;
    constexpr int EP = V * 64; // experts with padding
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    Sums<V> & z = *reinterpret_cast<Sums<V> *>(lds);
    float * part = z.part, * logit = z.logit;
    auto & xsq = z.xsq;
    auto & wsq = z.wsq;
    uint16_t * list = z.list;
    int & count = z.count;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, E = a.n_experts;
    const int row0 = blockIdx.x * 16, tiles = (E + 15) / 16, steps = a.dim >> 5; // (dim is a multiple of 32)
    const int KS = MW / tiles, t = wave % tiles, ks = wave / tiles;              // (waves past tiles KS have no steps)
    f32x4 acc = {0.f, 0.f, 0.f, 0.f}, nx = acc, nw = acc;
    // rows 0 .. 15 of x, then the experts' (past the last one that one again); 32 pieces of 16 bytes a row, exchanged by the row's low bits: 16
    // rows' pieces lie in different banks
    const int held = 16 + tiles * 16, bytes = held * 512, chunks = (steps + 7) / 8;
    const unsigned base = (unsigned) __builtin_amdgcn_readfirstlane((unsigned) (size_t) (__attribute__((address_space(3))) uint8_t *) lds);
    const auto fetch = [&](int c) { // two rows a copy
        const int k0 = c * 256, pieces = min(a.dim - k0, 256) / 8;
        for (int p = wave; p < held / 2; p += MW) {
            const int r = 2 * p + (lane >> 5), at = min((lane & 31) ^ (r & 15), pieces - 1); // (slots past the last piece are not read)
            const T * from = r < 16 ? static_cast<const T *>(a.x) + min(row0 + r, a.rows - 1) * a.x_stride
                                    : static_cast<const T *>(a.w) + (size_t) min(r - 16, E - 1) * a.dim;
            dma16(from + k0 + at * 8, base + (c & (a.buffers - 1)) * bytes + p * 1024);
        }
    };
    fetch(0);
    for (int c = 0; c < chunks; c++) {
        vm_drain();
        __syncthreads();
        if (a.buffers == 2 && c + 1 < chunks) fetch(c + 1);
        const int n8 = min(steps - c * 8, 8), s0 = ks < KS ? n8 * ks / KS : 0, s1 = ks < KS ? n8 * (ks + 1) / KS : 0;
        const uint8_t * at = lds + (c & (a.buffers - 1)) * bytes;
        for (int s = s0; s < s1; s++) {
            const int slot = ((4 * s + g) ^ n) * 16;
            const auto x = *reinterpret_cast<const typename Elem<DT>::Raw8 *>(at + n * 512 + slot);
            const auto w = *reinterpret_cast<const typename Elem<DT>::Raw8 *>(at + (16 + t * 16 + n) * 512 + slot);
            nx = mfma16<DT>(x, x, nx);
            acc = mfma16<DT>(w, x, acc);
            nw = mfma16<DT>(w, w, nw);
        }
        if (a.buffers == 1 && c + 1 < chunks) {
            __syncthreads();
            fetch(c + 1);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) count = 0;
    // lane n: row n, register r: expert 4 g + r; the norms lie on the diagonal
    const bool diagonal = g == n >> 2;
    const auto diag = [&](f32x4 v) { return n & 2 ? (n & 1 ? v[3] : v[2]) : n & 1 ? v[1] : v[0]; };
    *reinterpret_cast<f32x4 *>(part + (wave * 16 + n) * 16 + 4 * g) = acc;
    if (diagonal && ks < KS) wsq[ks][t * 16 + n] = diag(nw);
    if (diagonal && t == 0 && ks < KS) xsq[ks][n] = diag(nx);
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * EP; i += MW * 64) {
        const int r = i / EP, e = i % EP;
        float v = 0.f;
        if (e < E)
            for (int k = 0; k < KS; k++) v += part[(k * tiles + (e >> 4)) * 256 + r * 16 + (e & 15)];
        logit[i] = v;
        if (e < E && row0 + r < a.rows) a.logits[(size_t) (row0 + r) * E + e] = v;
    }
    // (the square of a NaN's expert is a NaN, which fmaxf leaves out: its logits are NaNs, in 64 bits too, and the others' bound is the others')
    float wmax = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) {
        float v = 0.f;
        if (lane * V + i < E)
            for (int k = 0; k < KS; k++) v += wsq[k][lane * V + i];
        wmax = fmaxf(wmax, v);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) wmax = fmaxf(wmax, shfl_xor(wmax, m));
    __syncthreads();
    // a row a wave: the experts that lie too close to each other
    const int most = min(E, a.top_k + 4), r = wave;
    float l[V];
#pragma unroll
    for (int i = 0; i < V; i++) l[i] = logit[r * EP + lane * V + i];
    float xs = 0.f;
    for (int k = 0; k < KS; k++) xs += xsq[k][r];
    // (a row of zeros, as of padding, has exact logits; squares and products below fp32's smallest may have become zeros)
    bool zero = false;
    if (xs == 0.f) {
        const T * xr = static_cast<const T *>(a.x) + min(row0 + r, a.rows - 1) * a.x_stride;
        unsigned some = 0;
        for (int k = lane * 8; k < a.dim; k += 512) some |= Elem<DT>::top8(Elem<DT>::raw8(xr + k));
        zero = !__any(some != 0);
    }
    const float lost = (float) a.dim * 0x1p-126f;
    const float near = zero ? 0.f : 2.f * ((float) (chunks * ((7 + KS) / KS) + 40) * 0x1p-22f * sqrtf(xs + lost) * sqrtf(wmax + lost) + lost); // (the bound on two errors; a wave's steps of a chunk are 8 / KS at most, rounded up)
    Chosen<V> c = route_choose<V>(a, l, most);
    const float v = c.logit, last = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), a.top_k - 1)) - near;
    const float up = __shfl_up(v, 1), down = __shfl_down(v, 1);
    // (NaNs count as close)
    const bool in = lane < most && !(v < last), close = in && near != 0.f && ((lane > 0 && !(up - v > near)) || (lane + 1 < most && !(v - down > near)));
    const bool all = most < E && near != 0.f && (__ballot(in) >> (most - 1) & 1), again = row0 + r < a.rows && (all || __ballot(close));
    if (again) {
        if (all) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (lane * V + i < E) list[atomicAdd(&count, 1)] = (uint16_t) (r * EP + lane * V + i);
        } else if (close) list[atomicAdd(&count, 1)] = (uint16_t) (r * EP + c.expert);
    }
    __syncthreads();
    for (int i = wave; i < count; i += MW) {
        const int at = __builtin_amdgcn_readfirstlane(list[i]), m = at / EP, e = at % EP;
        const T * xr = static_cast<const T *>(a.x) + (row0 + m) * a.x_stride, * wr = static_cast<const T *>(a.w) + (size_t) e * a.dim;
        double s = 0;
        for (int k = lane * 8; k < a.dim; k += 512) {
            float u[8], v[8];
            load8<DT>(xr + k, u);
            load8<DT>(wr + k, v);
#pragma unroll
            for (int j = 0; j < 8; j++) s = __builtin_fma((double) u[j], (double) v[j], s);
        }
        s = wave_sum(s);
        if (lane == 0) {
            logit[at] = (float) s;
            a.logits[(size_t) (row0 + m) * E + e] = (float) s;
        }
    }
    __syncthreads();
    if (row0 + r >= a.rows) return;
    if (again) {
#pragma unroll
        for (int i = 0; i < V; i++) l[i] = logit[r * EP + lane * V + i];
        c = route_choose<V>(a, l, a.top_k);
    }
    route_weights<V>(a, row0 + r, l, c);
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

// k_route_many's calls (4,096 rows of 2,048 x 63 experts: 29 us by k_route_logits and k_route_pick)
static bool many(const RouteArgs & a, int dtype, int wtype) {
    return a.rows >= MANY_ROWS && dtype == wtype && dtype != DT_F32 && a.dim % 32 == 0 && a.n_experts <= 256 && !a.bias && a.x_stride % 8 == 0 && (((size_t) a.x | (size_t) a.w) & 15) == 0;
}
template <int DT, int V> static hipError_t many(RouteArgs a, hipStream_t st) {
    static std::atomic<uint64_t> done;
    const size_t values = (size_t) (16 + (a.n_experts + 15) / 16 * 16) * 512;
    a.buffers = 2 * values <= 150 * 1024 ? 2 : 1;
    const size_t lds = std::max(values * a.buffers, sizeof(Sums<V>));
    const hipError_t e = allow_lds(k_route_many<DT, V>, lds, done);
    return e != hipSuccess ? e : launch(k_route_many<DT, V>, dim3((a.rows + 15) / 16), dim3(MW * 64), lds, st, a);
}
template <int DT> static hipError_t many(const RouteArgs & a, hipStream_t st) {
    const int v = (a.n_experts + 63) / 64;
    return v <= 1 ? many<DT, 1>(a, st) : v <= 2 ? many<DT, 2>(a, st) : many<DT, 4>(a, st);
}
hipError_t launch_route(const RouteArgs & a, int dtype, int wtype, hipStream_t st) {
    if (many(a, dtype, wtype)) return dtype == DT_F16 ? many<DT_F16>(a, st) : many<DT_BF16>(a, st);
    const hipError_t e = launch_logits(a, dtype, wtype, st);
    return e != hipSuccess ? e : launch_pick(a, st);
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
