// A mixture-of-experts layer with 4-bit weights for a few tokens: h = silu(G x) (U x) of every (token, expert) pair, then
// y[m] = sum over the row's experts of w D h.  Four kernels: x made ready and the pairs sorted by their experts (with a router also the choice), the
// gate's and the up projection's rows together, the down projection of every pair, and the sum over a row's experts in their order (no
// atomics in sums: the same bits every time); of a single row the last two in one.
//
// Workgroups stand for (columns, one of the experts that occur).  An expert has few tokens, so what counts is the way of its codes: from HBM,
// and from 4 bits to an operand.  Codes become int8 with four vector instructions for 8 of them (fp16 takes 13), so x is made integer
// too: an exponent for every block, and three int8 planes (22 bits of the block's largest power of two; int8 units are one plane as they
// are).  Two planes, 14 bits, are too few for 16-bit x as well: beside a value 256 times as large in its block they leave half of an fp16 layer's
// results another than the nearest (47 rows, 2 of 8 experts 4,096 x 8,192: 176 us with two, 215 with three; 8 rows of 8 of 128 small ones 62 and 63).
// The matrix instruction's sums are exact, the scales multiply them in fp32.
//
// A wave has two tiles of 16 weight rows, lane (n = lane & 15, g = lane >> 4) 16 bytes, a block of 32 codes of row n, a step.  The instruction
// contracts over all four lane groups, so blocks with scales of their own must not meet in it: the planes go in on a (block) diagonal,
// operand rows for lane groups whose blocks share a weight scale, zeros in the other groups.  Blocks of 32 values with scales of their own:
// four groups, 4 rows of planes each.  Weight groups of 64 or 128 values, and x with one exponent for as many: two lane groups or all
// four share a sum, 8 or 16 rows of planes go in at a time, and every sum is scaled once for 64 or 128 values.
#include "step_moe_plan.h"
#include "step_route_dev.h"

namespace qkv {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// the block of lane group g in step u of a run of 8 blocks: groups that share a sum have blocks of one weight group, and a lane's two steps
// have scales that lie next to each other
template <int SG> __device__ __forceinline__ int block_of(int g, int u) {
    return SG == 0 ? 2 * g + u : SG == 1 ? 4 * (g >> 1) + 2 * u + (g & 1) : 4 * u + g;
}
// the place in a row of 16 bytes of a block
template <int SG> __device__ __forceinline__ int piece(int block, int half) {
    const int b = block & 7, g = SG == 0 ? b >> 1 : SG == 1 ? 2 * (b >> 2) + (b & 1) : b & 3, u = SG == 0 ? b & 1 : SG == 1 ? b >> 1 & 1 : b >> 2;
    return ((block >> 3) * 4 + u * 2 + half) * 64 + g * 16;
}
__device__ __forceinline__ int piece(int sg, int block, int half) { return sg == 0 ? piece<0>(block, half) : sg == 1 ? piece<1>(block, half) : piece<2>(block, half); }

// values as integers: times `up`, a power of two that brings the largest to [2^21, 2^22), and the factor 1 / (16 up) of the products with
// codes 16 times as large
struct Fixed {
    float up, dx;
};
__device__ __forceinline__ Fixed fixed_of(unsigned top) {
    constexpr int S = 21;
    const int E = max((int) (top >> 23), 26);
    if (top >= 0x7f800000u) return Fixed{0.f, __builtin_nanf("")}; // an infinity or a NaN: the row's results are NaN
    return Fixed{__builtin_bit_cast(float, (unsigned) (254 + S - E) << 23), __builtin_bit_cast(float, (unsigned) (E - S - 4) << 23)};
}
// plane p of the integer v: its bits from 8 (2 - p) on as signed bytes
__device__ __forceinline__ void planes_split(int v, int (&q)[3]) {
#pragma unroll
    for (int p = 2; p > 0; p--) {
        q[p] = (int) (int8_t) v;
        v = (v - q[p]) >> 8;
    }
    q[0] = v;
}
__device__ __forceinline__ int to_fixed(float v, float up) { return up == 0.f ? 0 : (int) __builtin_rintf(v * up); } // (0 inf is a NaN)

// NT tiles of 16 weight rows: a tile's first row in scalars, the lane's in 32 bits behind it
template <int NT> struct Rows {
    const uint8_t * c[NT];
    const uint16_t * s[NT], * m[NT];
    unsigned vc[NT], vs[NT];
    // tile t: rows from `first` on of an expert's, rows past its last one (of n) that one again
    __device__ __forceinline__ void set(int t, const MoeWeights & w, int e, int n, int first, int nb, int gs) {
        const int f = min(first, n - 1), r = min((int) (threadIdx.x & 15), n - 1 - f);
        const size_t row = (size_t) e * n + f;
        c[t] = w.codes + row * (nb * 16);
        s[t] = w.scales + row * gs;
        m[t] = w.mins + row * gs;
        vc[t] = (unsigned) (r * nb * 16);
        vs[t] = (unsigned) (r * gs);
    }
};
// A run's codes and a window's scales in registers.  Scales come 32 of a row at a time (64 contiguous bytes; a lane's own of every run would
// fetch each cache line many times) and go through LDS of the wave's own.  Two runs are on their way: one alone leaves a wave waiting for memory.
template <int NT, bool MINS> struct Run {
    u32x4 c[2][NT][2];
    u32x4 s[NT], m[NT];
};
template <int GSH, int NT, bool MINS> __device__ __forceinline__ void load_window(const Rows<NT> & w, int nb, int R, Run<NT, MINS> & r) {
    const int g = threadIdx.x >> 4 & 3, gs = (nb + (1 << GSH) - 1) >> GSH, at = ((8 * R) >> GSH) + 8 * g;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        r.s[t] = w4_scales(w.s[t] + w.vs[t], gs, at);
        if constexpr (MINS) r.m[t] = w4_scales(w.m[t] + w.vs[t], gs, at);
    }
}
template <int SG, int NT> __device__ __forceinline__ void load_codes(const Rows<NT> & w, int nb, int R, int t, int u, u32x4 & c) {
    const int g = threadIdx.x >> 4 & 3; // (past the last block zeros of x, or of its factors)
    c = *reinterpret_cast<const u32x4 *>(w.c[t] + (w.vc[t] + (unsigned) min(8 * R + block_of<SG>(g, u), nb - 1) * 16));
}
// the first two of runs R .. last
template <int GSH, int SG, int NT, bool MINS> __device__ __forceinline__ Run<NT, MINS> load_runs(const Rows<NT> & w, int nb, int R, int last) {
    Run<NT, MINS> r;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int u = 0; u < 2; u++) load_codes<SG>(w, nb, R, t, u, r.c[0][t][u]);
    load_window<GSH>(w, nb, R, r);
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int u = 0; u < 2; u++) load_codes<SG>(w, nb, min(R + 1, last), t, u, r.c[1][t][u]);
    return r;
}

// adds the sums of the part p for nt tokens in LDS, at most TM, to acc.  in: the first two runs' codes and the first window of scales; those of the
// part q behind
template <int P, int GSH, int SG, int NT, int TM, bool MINS>
__device__ __forceinline__ void products(const Rows<NT> & w, Run<NT, MINS> & in, int nb, Part p, Part nx, const uint8_t * lds, const Lds & L, uint16_t * win, int tp, int nt, float (&acc)[NT][TM >> SG]) {
    const int r0 = p.r0, r1 = p.r1;
    constexpr int PR = op_rows(P), TL = lane_tokens(P), TG = group_of(P, SG);
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, m = n & ((4 << SG) - 1);
    const bool active = n >> (2 + SG) == g >> SG && m % PR < P;
    const int amask = active ? ~0 : 0, aoff = active ? (m / PR * P + m % PR) * L.row + g * 16 : L.zero, astep = TG * P * L.row & amask;
    const int first = (g & ((1 << SG) - 1)) * TL; // of a group's tokens, the first in the lane's sums
    const float * dx = reinterpret_cast<const float *>(lds + L.dx), * ds = reinterpret_cast<const float *>(lds + L.ds);
    const auto run = [&](int R, int buf) {
        const int next = R + 2 < r1 ? R + 2 : min(nx.r0 + buf, nx.r1 - 1);
        const int in_win = (R - r0) & ((4 << GSH) - 1);
        float sc[NT][2], mn[NT][2];
        const auto scales = [&](const uint16_t * p, float (&v)[2]) {
            if constexpr (SG == GSH) {
                const unsigned e = *reinterpret_cast<const unsigned *>(p + ((8 * in_win) >> GSH) + 2 * (g >> SG));
                v[0] = h2f_bits((uint16_t) e);
                v[1] = h2f_bits((uint16_t) (e >> 16));
            } else v[0] = v[1] = h2f_bits(p[(8 * in_win + 2 * g) >> GSH]);
        };
#pragma unroll
        for (int t = 0; t < NT; t++) {
            scales(win + (t * 16 + n) * WROW, sc[t]);
            if constexpr (MINS) scales(win + ((NT + t) * 16 + n) * WROW, mn[t]);
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            i32x4 b[NT][2];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    int t0, t1;
                    w4_bytes(in.c[buf][t][u][k], t0, t1);
                    b[t][k >> 1][2 * (k & 1)] = t0;
                    b[t][k >> 1][2 * (k & 1) + 1] = t1;
                }
            __builtin_amdgcn_sched_barrier(0); // the codes leave their registers, then those of a later run take them
#pragma unroll
            for (int t = 0; t < NT; t++) load_codes<SG>(w, nb, next, t, u, in.c[buf][t][u]);
            __builtin_amdgcn_sched_barrier(0);
            const uint8_t * ap = lds + (aoff + ((R - p.first) * 256 & amask)) + u * 128;
            const int at = ((8 * (R - p.first) + block_of<SG>(g, u)) >> SG) * tp + first;
#pragma unroll
            for (int q = 0; q < TM / TG; q++) {
                if (q * TG >= nt) continue;
                const i32x4 a0 = *reinterpret_cast<const i32x4 *>(ap), a1 = *reinterpret_cast<const i32x4 *>(ap + 64);
                ap += astep;
                i32x4 c[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    c[t] = i32x4{0, 0, 0, 0};
                    c[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, b[t][0], c[t], 0, 0, 0);
                    c[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, b[t][1], c[t], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < TL; i++) {
                    const float d = dx[at + q * TG + i];
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        float v;
                        if constexpr (P == 1) v = (float) c[t][i];
                        else v = __builtin_fmaf((float) ((c[t][0] << 8) + c[t][1]), 256.f, (float) c[t][2]);
                        float & s = acc[t][q * TL + i];
                        s = __builtin_fmaf(v, sc[t][u] * d, s);
                        if constexpr (MINS) s = __builtin_fmaf(mn[t][u], ds[at + q * TG + i], s);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
#pragma unroll 1
    for (int R = r0; R < r1; R += 2) {
        if (((R - r0) & ((4 << GSH) - 1)) == 0) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                *reinterpret_cast<u32x4 *>(win + (t * 16 + n) * WROW + 8 * g) = in.s[t];
                if constexpr (MINS) *reinterpret_cast<u32x4 *>(win + ((NT + t) * 16 + n) * WROW + 8 * g) = in.m[t];
            }
            asm volatile("" ::: "memory"); // (read below by other lanes and as another type)
            const bool more = R + (4 << GSH) < r1;
            if (more || nx.first != p.first) load_window<GSH>(w, nb, more ? R + (4 << GSH) : nx.r0, in);
        }
        run(R, 0);
        if (R + 1 < r1) run(R + 1, 1);
    }
}
// the wave's sums of nt tokens to red[tile][tp][16]: added over the lane groups that have the same token
template <int P, int SG, int NT, int TM> __device__ __forceinline__ void sums_out(float (&acc)[NT][TM >> SG], int tp, int nt, float * red) {
    constexpr int TL = lane_tokens(P), TG = group_of(P, SG);
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, first = (g & ((1 << SG) - 1)) * TL;
#pragma unroll
    for (int q = 0; q < TM / TG; q++) {
        if (q * TG >= nt) continue;
#pragma unroll
        for (int i = 0; i < TL; i++)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float v = acc[t][q * TL + i];
                if constexpr (SG == 0) v = quad_sum(v);
                if constexpr (SG == 1) v += shfl_xor(v, 32);
                if (g >> SG == 0 && q * TG + first + i < tp) red[(t * tp + q * TG + first + i) * 16 + n] = v;
            }
    }
}

// The experts that occur, those of more than LONG pairs first (their workgroups last longest), and the pairs that chose each (in any order: a
// pair's results do not depend on its place).  Choices that are no expert are left out.
constexpr int LONG = 8;
struct Lists {
    int count;
    uint16_t expert[ROUTE_MAX_EXPERTS], start[ROUTE_MAX_EXPERTS], pairs[ROUTE_MAX_EXPERTS], pair[MAX_PAIRS], row[MAX_PAIRS];
};

struct PrepArgs {
    MoeArgs a;
    RouteArgs r;
    int sg, rb; // of x: lane groups that share a sum are 1 << sg; bytes of a plane's row
};
constexpr int PREP = 1024; // threads

// The first workgroup: the choice (V experts a lane; 0: it is given) and its lists; the others: 8 values of x a thread
template <int XF, int V> __global__ __launch_bounds__(PREP) void k_moe_prep(PrepArgs d) {
    const MoeArgs & a = d.a;
    constexpr int P = planes_of(XF);
    const int nb = a.dim >> 5, nbp = padded(nb), tid = threadIdx.x;
    if (blockIdx.x == 0) {
        __shared__ int count[ROUTE_MAX_EXPERTS];
        __shared__ unsigned sums[PREP / 64];
        __shared__ int16_t chosen[MAX_PAIRS];
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, pairs = a.rows * a.top_k;
        count[tid] = 0;
        if constexpr (V > 0) {
            for (int row = wave; row < a.rows; row += PREP / 64) {
                const int e = route_pick<V>(d.r, row);
                if (lane < a.top_k) chosen[row * a.top_k + lane] = (int16_t) e;
            }
            __syncthreads();
        }
        int e = -1;
        if (tid < pairs) e = V > 0 ? chosen[tid] : a.ids[tid];
        if ((unsigned) e >= (unsigned) a.n_experts) e = -1;
        __syncthreads();
        if (e >= 0) atomicAdd(&count[e], 1);
        __syncthreads();
        // in front of expert tid: pairs (11 bits), experts that occur (11), experts of many pairs (10)
        const unsigned c = (unsigned) count[tid], v = c + (c ? 1u << 11 : 0) + (c > LONG ? 1u << 22 : 0);
        unsigned sum = v;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const unsigned o = __shfl_up(sum, m);
            if (lane >= m) sum += o;
        }
        if (lane == 63) sums[wave] = sum;
        __syncthreads();
        unsigned all = 0;
        for (int w = 0; w < PREP / 64; w++) {
            if (w == wave) sum += all;
            all += sums[w];
        }
        Lists * l = reinterpret_cast<Lists *>(a.lists);
        const int longs = (int) ((sum - v) >> 22), at = c > LONG ? longs : (int) (all >> 22) + (int) ((sum - v) >> 11 & 0x7ff) - longs, before = (int) ((sum - v) & 0x7ff);
        if (c) {
            l->expert[at] = (uint16_t) tid;
            l->start[at] = (uint16_t) before;
            l->pairs[at] = (uint16_t) c;
        }
        if (tid == 0) l->count = (int) (all >> 11 & 0x7ff);
        __syncthreads();
        count[tid] = before;
        __syncthreads();
        if (e >= 0) {
            const int to = atomicAdd(&count[e], 1);
            l->pair[to] = (uint16_t) tid;
            l->row[to] = (uint16_t) (tid / a.top_k);
        }
        return;
    }
    const int i = (blockIdx.x - 1) * PREP + tid, row = i / (nbp * 4), j = i - row * nbp * 4, block = j >> 2, qt = j & 3;
    if (row >= a.rows) return; // (whole blocks, and all blocks of an exponent, are in a wave)
    uint8_t * to = a.xq + (size_t) row * P * d.rb + piece(d.sg, block, qt >> 1) + 8 * (qt & 1);
    const size_t ndp = (size_t) (nbp >> d.sg);
    if constexpr (XF == W4_UNITS) {
        uint2 q = make_uint2(0, 0);
        float dd = 0.f, s = 0.f;
        if (block < nb) {
            const size_t unit = (size_t) row * nb + (block & ~1);
            q = *reinterpret_cast<const uint2 *>((block & 1 ? a.xb : a.xa) + (unit + (qt >> 1)) * 16 + 8 * (qt & 1));
            const uint16_t * m = a.xmeta + unit * 4;
            dd = h2f_bits(m[block & 1]);
            s = dd * (float) ((int) (int16_t) m[2 + (block & 1)] + (int) (int16_t) m[6 + (block & 1)]);
        }
        *reinterpret_cast<uint2 *>(to) = q;
        if (qt == 0) {
            a.xd[row * ndp + block] = dd * 0.0625f;
            a.xs[row * ndp + block] = s;
        }
    } else {
        float v[8], s = 0.f;
        typename Elem<XF>::Raw8 raw{};
        if (block < nb) raw = Elem<XF>::raw8(static_cast<const typename Elem<XF>::T *>(a.x) + row * a.x_stride + 32 * block + 8 * qt);
        unsigned top = Elem<XF>::top8(raw);
        Elem<XF>::open8(raw, v);
#pragma unroll
        for (int k = 0; k < 8; k++) s += v[k];
        // 4 << sg lanes an exponent
#pragma unroll
        for (int m = 1; m < 16; m <<= 1)
            if (m < 4 << d.sg) {
                top = max(top, shfl_xor_u(top, m));
                s += shfl_xor(s, m);
            }
        const Fixed f = fixed_of(top);
        unsigned out[P][2] = {};
#pragma unroll
        for (int k = 0; k < 8; k++) {
            int q[P];
            planes_split(to_fixed(v[k], f.up), q);
#pragma unroll
            for (int p = 0; p < P; p++) out[p][k >> 2] |= (unsigned) (q[p] & 255) << 8 * (k & 3);
        }
#pragma unroll
        for (int p = 0; p < P; p++) *reinterpret_cast<uint2 *>(to + (size_t) p * d.rb) = make_uint2(out[p][0], out[p][1]);
        if ((j & ((4 << d.sg) - 1)) == 0) {
            a.xd[row * ndp + (block >> d.sg)] = block < nb ? f.dx : 0.f;
            a.xs[row * ndp + (block >> d.sg)] = s;
        }
    }
}

__device__ __forceinline__ unsigned lds_address(const uint8_t * lds) {
    return (unsigned) __builtin_amdgcn_readfirstlane((unsigned) (size_t) (const __attribute__((address_space(3))) uint8_t *) lds);
}
// the planes, factors and sums of nt tokens, lane t's `at` the place of the t-th, into LDS: of runs c0 .. c0 + n - 1 (rows of `row` bytes, nd factors, ng of
// them in use)
template <int P, bool MINS, int W = WAVES>
__device__ __forceinline__ void stage(const uint8_t * q, const float * d, const float * s, int row, int nd, int ng, int c0, int n, int sg, uint8_t * lds, const Lds & L, int tp, int nt, int at) {
    const unsigned base = lds_address(lds);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, bytes = n * 256, per = (bytes + 1023) >> 10, d0 = c0 * 8 >> sg, dn = n * 8 >> sg;
    float * dx = reinterpret_cast<float *>(lds + L.dx), * ds = reinterpret_cast<float *>(lds + L.ds);
    int c = wave;
    for (int t = 0; t < nt; t++) { // 1 KiB a copy, the waves in turn
        const uint8_t * from = q + (size_t) (unsigned) __builtin_amdgcn_readlane(at, t) * (P * row) + c0 * 256;
#pragma unroll
        for (int p = 0; p < P; p++, c -= per)
            for (; c < per; c += W)
                if (c * 1024 + lane * 16 < bytes) dma16(from + (p * row + c * 1024 + lane * 16), base + (t * P + p) * L.row + c * 1024);
    }
    for (int k = tid; k < dn; k += W * 64)
        for (int t0 = 0; t0 < nt; t0 += 4) { // (four loads, then their values)
            float v[4], w[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const size_t i = (size_t) (unsigned) __builtin_amdgcn_readlane(at, min(t0 + u, nt - 1)) * nd + d0 + k;
                v[u] = d[i];
                if (MINS) w[u] = s[i];
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (t0 + u < nt) {
                    dx[k * tp + t0 + u] = d0 + k < ng ? v[u] : 0.f; // (of blocks past the last one: nothing)
                    if (MINS) ds[k * tp + t0 + u] = d0 + k < ng ? w[u] : 0.f;
                }
        }
    vm_drain();
}
__device__ __forceinline__ void zero_pieces(uint8_t * lds, const Lds & L) {
    if (threadIdx.x < 64) reinterpret_cast<unsigned *>(lds + L.zero)[threadIdx.x] = 0;
}

// The gate and the up projection: a workgroup has 16 CG inner columns of an expert, its waves (16 columns of both, a KS-th of dim), CG KS = WAVES.
// SG: lane groups that share a sum of x; SH: those of the down projection, whose x (h) this kernel leaves as planes.
template <int P, int GSH, int SH, int TM, bool MINS> __global__ __launch_bounds__(WAVES * 64, PER_CU) void k_moe_up(MoeArgs a) {
    constexpr int SG = P == 1 ? 0 : GSH;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const Lists * l = reinterpret_cast<const Lists *>(a.lists);
    if ((int) blockIdx.y >= l->count) return;
    const int e = l->expert[blockIdx.y], p0 = l->start[blockIdx.y], cnt = l->pairs[blockIdx.y];
    const int nb = a.dim >> 5, nbp = padded(nb), runs = nbp >> 3, tp = a.tp_up;
    const Lds L = lds_of(P, SG, a.cr_up, tp, MINS);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // each wave's window of scales, then its sums: [KS][CG][2][tp][16]
    constexpr int WB = win_bytes(2, MINS) / 4;
    float * red = reinterpret_cast<float *>(lds + L.end);
    uint16_t * win = reinterpret_cast<uint16_t *>(red + wave * WB);
    const int KS = 1 << a.ks_up, CG = WAVES >> a.ks_up, cg = wave & (CG - 1), ks = wave / CG;
    const int gs = (nb + (1 << GSH) - 1) >> GSH, c0 = blockIdx.x * 16 * CG, chunks = (runs + a.cr_up - 1) / a.cr_up;
    Rows<2> w; // (columns past the last one: zeros below)
    w.set(0, a.up, 2 * e, a.inner, c0 + cg * 16, nb, gs);
    w.set(1, a.up, 2 * e + 1, a.inner, c0 + cg * 16, nb, gs);
    zero_pieces(lds, L);
    for (int t0 = 0; t0 < cnt; t0 += tp) {
        const int nt = min(tp, cnt - t0);
        const int at = l->row[p0 + t0 + min((int) (threadIdx.x & 63), nt - 1)];
        Part part = part_of(runs, a.cr_up, 0, ks, a.ks_up);
        Run<2, MINS> in = load_runs<GSH, SG, 2, MINS>(w, nb, part.r0, part.r1 - 1); // (on its way while x is made ready)
        float acc[2][TM >> SG];
#pragma unroll
        for (int i = 0; i < TM >> SG; i++) acc[0][i] = acc[1][i] = 0.f;
        for (int c = 0; c < chunks; c++) {
            const Part next = c + 1 < chunks ? part_of(runs, a.cr_up, c + 1, ks, a.ks_up) : Part{part.first, part.r1 - 1, part.r1}; // (behind the last run that one again, unused)
            if (t0 + c) __syncthreads();
            stage<P, MINS>(a.xq, a.xd, a.xs, plane_bytes(nb), nbp >> SG, (nb + (1 << SG) - 1) >> SG, part.first, min(a.cr_up, runs - part.first), SG, lds, L, tp, nt, at);
            __syncthreads();
            products<P, GSH, SG, 2, TM, MINS>(w, in, nb, part, next, lds, L, win, tp, nt, acc);
            part = next;
        }
        sums_out<P, SG, 2, TM>(acc, tp, nt, red + (ks * CG + cg) * WB);
        __syncthreads();
        // four columns of a token a thread, 8 << SH threads for the values of an exponent of h
        for (int j = threadIdx.x; j < nt * CG * 4; j += WAVES * 64) {
            const int i = j >> (WAVES_LOG + 2 - a.ks_up), col = (j & (CG * 4 - 1)) * 4, c = c0 + col;
            f32x4 gt = {0.f, 0.f, 0.f, 0.f}, up = gt, h;
            for (int k = 0; k < KS; k++) {
                const float * p = red + ((k * CG + (col >> 4)) * WB + i * 16 + (col & 15));
                gt += *reinterpret_cast<const f32x4 *>(p);
                up += *reinterpret_cast<const f32x4 *>(p + tp * 16);
            }
            unsigned top = 0;
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                h[k] = c < a.inner ? gt[k] / (1.f + expf(-gt[k])) * up[k] : 0.f; // (inner is a multiple of 32)
                const float hk = h[k]; // (a bit cast of a vector's element itself takes the first one)
                top = max(top, __builtin_bit_cast(unsigned, hk) & 0x7fffffffu);
                s += hk;
            }
#pragma unroll
            for (int m = 1; m < 8 << SH; m <<= 1) {
                top = max(top, shfl_xor_u(top, m));
                if (MINS) s += shfl_xor(s, m);
            }
            const Fixed f = fixed_of(top);
            unsigned out[HP] = {};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                int q[HP];
                planes_split(to_fixed(h[k], f.up), q);
#pragma unroll
                for (int p = 0; p < HP; p++) out[p] |= (unsigned) (q[p] & 255) << 8 * k;
            }
            const int nbi = padded(a.inner >> 5), block = c >> 5, pair = l->pair[p0 + t0 + i];
            if (block >= nbi) continue;
            uint8_t * to = a.hq + (size_t) pair * HP * plane_bytes(nbi) + piece<SH>(block, c >> 4 & 1) + (c & 15);
#pragma unroll
            for (int p = 0; p < HP; p++) *reinterpret_cast<unsigned *>(to + (size_t) p * plane_bytes(nbi)) = out[p];
            if ((c & ((32 << SH) - 1)) == 0) {
                a.hd[(size_t) pair * (nbi >> SH) + (block >> SH)] = f.dx;
                if (MINS) a.hs[(size_t) pair * (nbi >> SH) + (block >> SH)] = s;
            }
        }
    }
}

// the down projection of every pair: waves (32 columns, a KS-th of inner)
template <int GSH, int SG, int TM, bool MINS> __global__ __launch_bounds__(WAVES * 64, PER_CU) void k_moe_down(MoeArgs a) {
    constexpr int P = HP;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const Lists * l = reinterpret_cast<const Lists *>(a.lists);
    if ((int) blockIdx.y >= l->count) return;
    const int e = l->expert[blockIdx.y], p0 = l->start[blockIdx.y], cnt = l->pairs[blockIdx.y];
    const int nb = a.inner >> 5, nbp = padded(nb), runs = nbp >> 3, tp = a.tp_down;
    const Lds L = lds_of(P, SG, a.cr_down, tp, MINS);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // each wave's window of scales, then its sums: [KS][CG][2][tp][16]
    constexpr int WB = win_bytes(2, MINS) / 4;
    float * red = reinterpret_cast<float *>(lds + L.end);
    uint16_t * win = reinterpret_cast<uint16_t *>(red + wave * WB);
    const int KS = 1 << a.ks_down, CG = WAVES >> a.ks_down, cg = wave & (CG - 1), ks = wave / CG;
    const int gs = (nb + (1 << GSH) - 1) >> GSH, c0 = blockIdx.x * CG * 32, chunks = (runs + a.cr_down - 1) / a.cr_down;
    Rows<2> w; // (columns past the last one: not stored)
    w.set(0, a.down, e, a.dim, c0 + cg * 32, nb, gs);
    w.set(1, a.down, e, a.dim, c0 + cg * 32 + 16, nb, gs);
    zero_pieces(lds, L);
    for (int t0 = 0; t0 < cnt; t0 += tp) {
        const int nt = min(tp, cnt - t0);
        const int at = l->pair[p0 + t0 + min((int) (threadIdx.x & 63), nt - 1)];
        Part part = part_of(runs, a.cr_down, 0, ks, a.ks_down);
        Run<2, MINS> in = load_runs<GSH, SG, 2, MINS>(w, nb, part.r0, part.r1 - 1); // (on its way while x is made ready)
        float acc[2][TM >> SG];
#pragma unroll
        for (int i = 0; i < TM >> SG; i++) acc[0][i] = acc[1][i] = 0.f;
        for (int c = 0; c < chunks; c++) {
            const Part next = c + 1 < chunks ? part_of(runs, a.cr_down, c + 1, ks, a.ks_down) : Part{part.first, part.r1 - 1, part.r1}; // (behind the last run that one again, unused)
            if (t0 + c) __syncthreads();
            stage<P, MINS>(a.hq, a.hd, a.hs, plane_bytes(nb), nbp >> SG, (nb + (1 << SG) - 1) >> SG, part.first, min(a.cr_down, runs - part.first), SG, lds, L, tp, nt, at);
            __syncthreads();
            products<P, GSH, SG, 2, TM, MINS>(w, in, nb, part, next, lds, L, win, tp, nt, acc);
            part = next;
        }
        sums_out<P, SG, 2, TM>(acc, tp, nt, red + (ks * CG + cg) * WB);
        __syncthreads();
        for (int j = threadIdx.x; j < nt * CG * 8; j += WAVES * 64) {
            const int i = j >> (WAVES_LOG + 3 - a.ks_down), col = (j & (CG * 8 - 1)) * 4, c = c0 + col;
            if (c >= a.dim) continue;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < KS; k++) v += *reinterpret_cast<const f32x4 *>(red + ((k * CG + (col >> 5)) * WB + ((col >> 4 & 1) * tp + i) * 16 + (col & 15)));
            *reinterpret_cast<f32x4 *>(a.out + (size_t) l->pair[p0 + t0 + i] * a.dim + c) = v;
        }
    }
}

// The down projection of a single row and the sum over its experts, in one launch: a workgroup has 16 NT columns of all of them, its waves (an expert,
// a part of inner).  Tokens in LDS are the row's pairs; no list is needed.  A layer's row, 8 of 128 experts of 2,048 x 768: 26.3 us, 28.6 with k_moe_down and
// k_moe_sum; 2 of 8 of 5,120 x 6,144 in fp32: 45 and 49.
template <int GSH, int SG, int NT, bool MINS, int YT> __global__ __launch_bounds__(OW * 64) void k_moe_down_one(MoeArgs a) {
    constexpr int P = HP, TG = group_of(P, SG), WB = win_bytes(NT, MINS);
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c0 = blockIdx.x * 16 * NT;
    const int nb = a.inner >> 5, nbp = padded(nb), runs = nbp >> 3, gs = (nb + (1 << GSH) - 1) >> GSH, tp = a.top_k + TG;
    const Lds L = lds_of(P, SG, runs, tp, MINS);
    uint16_t * win = reinterpret_cast<uint16_t *>(lds + L.end + wave * WB);
    float * red = reinterpret_cast<float *>(lds + L.end + OW * WB); // [OW][NT][16]
    const int j = wave >> a.ks_one, ks = wave & ((1 << a.ks_one) - 1), e = j < a.top_k ? __builtin_amdgcn_readfirstlane(a.ids[min(j, a.top_k - 1)]) : -1;
    const bool on = (unsigned) e < (unsigned) a.n_experts;
    Rows<NT> w;
    Run<NT, MINS> in;
    const Part part = part_of(runs, runs, 0, ks, a.ks_one);
    if (on) {
#pragma unroll
        for (int t = 0; t < NT; t++) w.set(t, a.down, e, a.dim, c0 + 16 * t, nb, gs);
        in = load_runs<GSH, SG, NT, MINS>(w, nb, part.r0, part.r1 - 1);
    }
    zero_pieces(lds, L);
    stage<P, MINS, OW>(a.hq, a.hd, a.hs, plane_bytes(nb), nbp >> SG, (nb + (1 << SG) - 1) >> SG, 0, runs, SG, lds, L, tp, a.top_k, lane);
    __syncthreads();
    if (on) {
        // its pair's planes come first; those behind them take part in the instruction, and their sums are not used
        const int off = j * P * L.row;
        Lds l = L;
        l.zero -= off;
        l.dx += 4 * j - off;
        l.ds += 4 * j - off;
        float acc[NT][TG >> SG];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < TG >> SG; i++) acc[t][i] = 0.f;
        products<P, GSH, SG, NT, TG, MINS>(w, in, nb, part, Part{part.first, part.r1 - 1, part.r1}, lds + off, l, win, tp, 1, acc);
        sums_out<P, SG, NT, TG>(acc, 1, 1, red + wave * NT * 16);
    }
    __syncthreads();
    if (threadIdx.x >= 16 * NT) return;
    float v = 0.f;
    for (int p = 0; p < a.top_k; p++) {
        if ((unsigned) a.ids[p] >= (unsigned) a.n_experts) continue;
        float o = 0.f;
        for (int k = 0; k < 1 << a.ks_one; k++) o += red[((p << a.ks_one) + k) * NT * 16 + threadIdx.x];
        v = __builtin_fmaf(a.weights[p], o, v);
    }
    static_cast<typename Elem<YT>::T *>(a.y)[c0 + threadIdx.x] = Elem<YT>::down(v);
}

// y[m] = sum over the row's places, in order, of w out
template <int YT> __global__ __launch_bounds__(256) void k_moe_sum(MoeArgs a) {
    const int row = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (c >= a.dim) return; // (dim is a multiple of 32)
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < a.top_k; j++) {
        const int pair = row * a.top_k + j;
        if ((unsigned) a.ids[pair] >= (unsigned) a.n_experts) continue;
        const float w = a.weights[pair];
        const f32x4 o = *reinterpret_cast<const f32x4 *>(a.out + (size_t) pair * a.dim + c);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __builtin_fmaf(w, o[i], v[i]);
    }
    typename Elem<YT>::T * y = static_cast<typename Elem<YT>::T *>(a.y) + row * a.y_stride + c;
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = Elem<YT>::down(v[i]);
}

template <int P, int GSH, int SH, int TM, bool MINS> hipError_t up(const MoeArgs & a, int slots, hipStream_t st) {
    constexpr int SG = P == 1 ? 0 : GSH;
    static std::atomic<uint64_t> done;
    const size_t lds = lds_bytes(a, P, SG, a.cr_up, a.tp_up);
    const hipError_t e = allow_lds(k_moe_up<P, GSH, SH, TM, MINS>, lds, done);
    const int cols = 16 * (WAVES >> a.ks_up);
    return e != hipSuccess ? e : launch(k_moe_up<P, GSH, SH, TM, MINS>, dim3((a.inner + cols - 1) / cols, slots), dim3(WAVES * 64), lds, st, a);
}
template <int GSH, int SG, int TM, bool MINS> hipError_t down(const MoeArgs & a, int slots, hipStream_t st) {
    static std::atomic<uint64_t> done;
    const size_t lds = lds_bytes(a, HP, SG, a.cr_down, a.tp_down);
    const hipError_t e = allow_lds(k_moe_down<GSH, SG, TM, MINS>, lds, done);
    const int cols = 32 * (WAVES >> a.ks_down);
    return e != hipSuccess ? e : launch(k_moe_down<GSH, SG, TM, MINS>, dim3((a.dim + cols - 1) / cols, slots), dim3(WAVES * 64), lds, st, a);
}
template <int GSH, int SG, int NT, bool MINS, int YT> hipError_t down_one(const MoeArgs & a, hipStream_t st) {
    static std::atomic<uint64_t> done;
    const size_t lds = one_lds(a, HP, SG, NT);
    const hipError_t e = allow_lds(k_moe_down_one<GSH, SG, NT, MINS, YT>, lds, done);
    return e != hipSuccess ? e : launch(k_moe_down_one<GSH, SG, NT, MINS, YT>, dim3(a.dim / (16 * NT)), dim3(OW * 64), lds, st, a);
}
template <int XF, int GSH, int SH, bool MINS> hipError_t run(const MoeArgs & a, hipStream_t st) {
    constexpr int YT = XF == W4_UNITS ? DT_F32 : XF;
    const int slots = std::min(a.n_experts, a.rows * a.top_k);
    hipError_t e = a.tp_up <= 8 ? up<planes_of(XF), GSH, SH, 8, MINS>(a, slots, st) : up<planes_of(XF), GSH, SH, 16, MINS>(a, slots, st);
    if (e != hipSuccess) return e;
    // (a workgroup a CU: 16 columns, or 32 where those would be more)
    if (one_row(a)) return a.dim <= 256 * 16 ? down_one<GSH, SH, 1, MINS, YT>(a, st) : down_one<GSH, SH, 2, MINS, YT>(a, st);
    e = a.tp_down <= 8 ? down<GSH, SH, 8, MINS>(a, slots, st) : down<GSH, SH, 16, MINS>(a, slots, st);
    if (e != hipSuccess) return e;
    return launch(k_moe_sum<YT>, dim3((a.dim + 1023) / 1024, a.rows), dim3(256), 0, st, a);
}
template <int XF, int GSH, bool MINS> hipError_t run(const MoeArgs & a, hipStream_t st) {
    if constexpr (GSH == 0) return run<XF, 0, 0, MINS>(a, st);
    else return a.ks_up == 0 ? run<XF, GSH, 1, MINS>(a, st) : run<XF, GSH, 0, MINS>(a, st);
}
template <int XF, bool MINS> hipError_t run(const MoeArgs & a, hipStream_t st) {
    return a.gsh == 0 ? run<XF, 0, MINS>(a, st) : a.gsh == 1 ? run<XF, 1, MINS>(a, st) : run<XF, 2, MINS>(a, st);
}
template <int XF> hipError_t run(const MoeArgs & a, hipStream_t st) { return a.up.mins ? run<XF, true>(a, st) : run<XF, false>(a, st); }

} // namespace

long long moe_plan(MoeArgs & a, int xform, uint8_t * ws) {
    const int P = planes_of(xform), nbx = a.dim / 32, nbi = a.inner / 32;
    const long long rows = std::min(a.rows, MOE_ROWS), pairs = rows * a.top_k;
    long long at = 0;
    const auto take = [&](long long bytes) {
        uint8_t * p = ws + at;
        at += (bytes + 255) & ~255ll;
        return p;
    };
    a.lists = take(sizeof(Lists));
    a.hq = take(pairs * HP * plane_bytes(nbi));
    a.hd = reinterpret_cast<float *>(take(pairs * padded(nbi) * 4));
    a.hs = reinterpret_cast<float *>(take(a.up.mins ? pairs * padded(nbi) * 4 : 0));
    // x is not used any more once the experts' outputs are written
    const long long here = at;
    a.xq = take(rows * P * plane_bytes(nbx));
    a.xd = reinterpret_cast<float *>(take(rows * padded(nbx) * 4));
    a.xs = reinterpret_cast<float *>(take(rows * padded(nbx) * 4));
    const long long x_end = at;
    at = here;
    a.out = reinterpret_cast<float *>(take(pairs * a.dim * 4));
    return std::max(at, x_end);
}

template <int XF> static hipError_t prep(const MoeArgs & a, const RouteArgs * route, hipStream_t st) {
    constexpr int P = planes_of(XF);
    const int nb = a.dim / 32, threads = a.rows * padded(nb) * 4;
    const PrepArgs d{a, route ? *route : RouteArgs{}, P == 1 ? 0 : a.gsh, plane_bytes(nb)};
    const dim3 grid(1 + (threads + PREP - 1) / PREP), block(PREP);
    if (!route) return launch(k_moe_prep<XF, 0>, grid, block, 0, st, d);
    if constexpr (XF != W4_UNITS) {
        const int v = (a.n_experts + 63) / 64;
        return v <= 2 ? launch(k_moe_prep<XF, 2>, grid, block, 0, st, d) : launch(k_moe_prep<XF, 4>, grid, block, 0, st, d);
    }
    return hipErrorInvalidValue; // (a router takes plain rows)
}

hipError_t launch_moe(const MoeArgs & all, int xform, const RouteArgs * route, hipStream_t st) {
    const int xs = xform == DT_F32 ? 4 : 2, ys = xform == DT_F16 || xform == DT_BF16 ? 2 : 4, nb = all.dim / 32;
    for (int row = 0; row < all.rows; row += MOE_ROWS) {
        MoeArgs a = all;
        a.rows = std::min(MOE_ROWS, all.rows - row);
        a.ids += (size_t) row * a.top_k;
        a.weights += (size_t) row * a.top_k;
        a.y = static_cast<char *>(a.y) + row * a.y_stride * ys;
        if (xform == W4_UNITS) {
            a.xa += (size_t) row * nb * 16;
            a.xb += (size_t) row * nb * 16;
            a.xmeta += (size_t) row * nb * 4;
        } else a.x = static_cast<const char *>(a.x) + row * a.x_stride * xs;
        split_work(a, xform);
        if (!plan_holds(a, xform)) return hipErrorInvalidConfiguration; // (never: every shape that the entry points take has such a plan)
        hipError_t e = xform == W4_UNITS ? prep<W4_UNITS>(a, route, st) : xform == DT_F32 ? prep<DT_F32>(a, route, st) : xform == DT_F16 ? prep<DT_F16>(a, route, st) : prep<DT_BF16>(a, route, st);
        if (e != hipSuccess) return e;
        e = xform == W4_UNITS ? run<W4_UNITS>(a, st) : xform == DT_F32 ? run<DT_F32>(a, st) : xform == DT_F16 ? run<DT_F16>(a, st) : run<DT_BF16>(a, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

} // namespace qkv
