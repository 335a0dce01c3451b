// A mixture-of-experts layer with 4-bit weights for a few tokens: h = silu(G x) (U x) of every (token, expert) pair, then
// y[m] = sum over the row's experts of w D h.  Three kernels: the gate's and the up projection's rows together, the down projection of every
// pair, and the sum over a row's experts in their order (no atomics: the same bits every time); where the pairs are few the last two are
// one.
//
// Workgroups stand for (columns, one of the experts that occur); each finds its expert and the pairs that chose it in the rows'
// choices itself.  An expert has few tokens, so what counts is the way of its codes: from HBM, and from 4 bits to an operand.  Codes
// become int8 with four vector instructions for 8 of them (fp16 takes 13), so x is made integer too: an exponent for every block, and two
// or three int8 planes (14 bits of the block's largest power of two for 16-bit x, 22 for fp32; int8 units are one plane as
// they are).  The matrix instruction's sums are exact, the scales multiply them in fp32.
//
// A wave has two tiles of 16 weight rows, lane (n = lane & 15, g = lane >> 4) 16 bytes, a block of 32 codes of row n, a step.  The instruction
// contracts over all four lane groups, so blocks with scales of their own must not meet in it: the planes go in on a (block) diagonal,
// operand rows for lane groups whose blocks share a weight scale, zeros in the other groups.  Blocks of 32 values with scales of their own:
// four groups, 4 rows of planes each.  Weight groups of 64 or 128 values, and x with one exponent for as many: two lane groups or all
// four share a sum, 8 or 16 rows of planes go in at a time, and every sum is scaled once for 64 or 128 values.
#include "step_dev.h"
#include "step_mix_launch.h"

#include <algorithm>

namespace qkv {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32_u2 __attribute__((aligned(2)));

constexpr int MAX_PAIRS = MOE_ROWS * ROUTE_MAX_TOP;
constexpr int WAVES = 8;

constexpr int planes_of(int xform) { return xform == W4_UNITS ? 1 : xform == DT_F32 ? 3 : 2; }
constexpr int inner_planes(int xform) { return xform == DT_F16 || xform == DT_BF16 ? 2 : 3; } // (y is fp32 else)
// operand rows of a token (three planes: the fourth stays zero), tokens in a lane's sums of an instruction, tokens of an instruction; sg: lane
// groups that share a sum are 1 << sg
constexpr int op_rows(int P) { return P == 3 ? 4 : P; }
constexpr int lane_tokens(int P) { return 4 / op_rows(P); }
constexpr int group_of(int P, int sg) { return lane_tokens(P) << sg; }

// LDS of a pass: x as planes, token t's plane p is row t P + p: [runs of 8 blocks][u][half][rows][64 bytes: 16 of each lane group's block];
// where more than four rows go in for a group, the groups' places are exchanged every four rows (their pieces lie in different banks); then zeros for the operand's
// other lanes, per 32 << sg values the tokens' factors, and with minimums the tokens' sums
struct Lds {
    int step, zero, dx, ds, end; // bytes of all rows' 64; offsets
};
__host__ __device__ __forceinline__ constexpr Lds lds_of(int P, int sg, int nbp, int tp, bool mins) {
    Lds l{};
    l.step = tp * P * 64;
    l.zero = (nbp >> 1) * l.step;
    l.dx = l.zero + l.step + 64; // (the operand's offsets within a step go for the zeros too)
    l.ds = l.dx + (nbp >> sg) * tp * 4;
    l.end = mins ? l.ds + (nbp >> sg) * tp * 4 : l.ds;
    return l;
}
__host__ __device__ __forceinline__ constexpr int padded(int blocks) { return (blocks + 7) & ~7; }
// the block of lane group g in step u of a run of 8 blocks: groups that share a sum have blocks of one weight group, and a lane's two steps
// have scales that lie next to each other
template <int SG> __device__ __forceinline__ int block_of(int g, int u) {
    return SG == 0 ? 2 * g + u : SG == 1 ? 4 * (g >> 1) + 2 * u + (g & 1) : 4 * u + g;
}
// 16 bytes of a block: its place among a row's 64-byte pieces, and its group in it
template <int SG> __device__ __forceinline__ int piece_of(int block, int half) {
    const int b = block & 7, u = SG == 0 ? b & 1 : SG == 1 ? b >> 1 & 1 : b >> 2;
    return (block >> 3) * 4 + u * 2 + half;
}
template <int SG> __device__ __forceinline__ int group_in(int block) {
    const int b = block & 7;
    return SG == 0 ? b >> 1 : SG == 1 ? 2 * (b >> 2) + (b & 1) : b & 3;
}
template <int SG> __device__ __forceinline__ int turn(int row, int g) { return SG == 0 ? g : (g ^ (row >> 2)) & 3; }
template <int SG> __device__ __forceinline__ int place(int row, int g) { return row * 64 + turn<SG>(row, g) * 16; }

// values as integers: times `up`, a power of two that brings the largest to [2^13, 2^14) (three planes: [2^21, 2^22)), and the
// factor 1 / (16 up) of the products with codes 16 times as large
struct Fixed {
    float up, dx;
};
template <int P> __device__ __forceinline__ Fixed fixed_of(unsigned top) {
    constexpr int S = P == 3 ? 21 : 13;
    const int E = max((int) (top >> 23), 26);
    if (top >= 0x7f800000u) return Fixed{0.f, __builtin_nanf("")}; // an infinity or a NaN: the row's results are NaN
    return Fixed{__builtin_bit_cast(float, (unsigned) (254 + S - E) << 23), __builtin_bit_cast(float, (unsigned) (E - S - 4) << 23)};
}
// plane p of P of the integer v: its bits from 8 (P - 1 - p) on as signed bytes
template <int P> __device__ __forceinline__ void planes_split(int v, int (&q)[P]) {
#pragma unroll
    for (int p = P - 1; p > 0; p--) {
        q[p] = (int) (int8_t) v;
        v = (v - q[p]) >> 8;
    }
    q[0] = v;
}
template <int P> __device__ __forceinline__ int to_fixed(float v, float up) { return up == 0.f ? 0 : (int) __builtin_rintf(v * up); } // (0 inf is a NaN)

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
// a run's codes and scales in registers
template <int NT, bool MINS> struct Run {
    u32x4 c[NT][2];
    unsigned s[NT], m[NT]; // of the two steps (groups of more than 32 without a shared sum: one)
};
template <int GSH, int SG> __device__ __forceinline__ unsigned run_scales(const uint16_t * p, unsigned v, int gs, int R, int g) {
    const int i = ((8 * R) >> GSH) + (SG == GSH ? 2 * (g >> SG) : (2 * g) >> GSH);
    if constexpr (SG != GSH) return p[v + (unsigned) min(i, gs - 1)];
    if ((8 * R + 8) >> GSH <= gs) return *reinterpret_cast<const u32_u2 *>(p + (v + (unsigned) i));
    return p[v + (unsigned) min(i, gs - 1)] | (unsigned) p[v + (unsigned) min(i + 1, gs - 1)] << 16;
}
template <int GSH, int SG, int NT, bool MINS> __device__ __forceinline__ Run<NT, MINS> load_run(const Rows<NT> & w, int nb, int R) {
    const int g = threadIdx.x >> 4 & 3, gs = (nb + (1 << GSH) - 1) >> GSH;
    Run<NT, MINS> r;
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int u = 0; u < 2; u++) r.c[t][u] = *reinterpret_cast<const u32x4 *>(w.c[t] + (w.vc[t] + (unsigned) min(8 * R + block_of<SG>(g, u), nb - 1) * 16)); // (past the last block zeros of x, or of its factors)
        r.s[t] = run_scales<GSH, SG>(w.s[t], w.vs[t], gs, R, g);
        if constexpr (MINS) r.m[t] = run_scales<GSH, SG>(w.m[t], w.vs[t], gs, R, g);
    }
    return r;
}

// the sums of runs r0 .. r1 - 1 (in: the first one's codes) for nt tokens in LDS, at most TM
template <int P, int GSH, int SG, int NT, int TM, bool MINS>
__device__ __forceinline__ void products(const Rows<NT> & w, Run<NT, MINS> in, int nb, int r0, int r1, const uint8_t * lds, const Lds & L, int tp, int nt, float (&acc)[NT][TM >> SG]) {
    constexpr int PR = op_rows(P), TL = lane_tokens(P), TG = group_of(P, SG);
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, m = n & ((4 << SG) - 1), gs = (nb + (1 << GSH) - 1) >> GSH;
    const bool active = n >> (2 + SG) == g >> SG && m % PR < P;
    const int row = m / PR * P + m % PR;
    const int first = (g & ((1 << SG) - 1)) * TL; // of a group's tokens, the first in the lane's sums
    const float * dx = reinterpret_cast<const float *>(lds + L.dx), * ds = reinterpret_cast<const float *>(lds + L.ds);
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < TM >> SG; i++) acc[t][i] = 0.f;
#pragma unroll 1
    for (int R = r0; R < r1; R++) {
        const int next = min(R + 1, r1 - 1); // (behind the last run that one again, unused)
        float sc[NT][2], mn[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                sc[t][u] = h2f_bits((uint16_t) (in.s[t] >> (SG == GSH ? 16 * u : 0)));
                if constexpr (MINS) mn[t][u] = h2f_bits((uint16_t) (in.m[t] >> (SG == GSH ? 16 * u : 0)));
            }
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            i32x4 b[NT][2];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    int t0, t1;
                    w4_bytes(in.c[t][u][k], t0, t1);
                    b[t][k >> 1][2 * (k & 1)] = t0;
                    b[t][k >> 1][2 * (k & 1) + 1] = t1;
                }
            __builtin_amdgcn_sched_barrier(0); // the codes leave their registers, then the next run's take them
#pragma unroll
            for (int t = 0; t < NT; t++) {
                in.c[t][u] = *reinterpret_cast<const u32x4 *>(w.c[t] + (w.vc[t] + (unsigned) min(8 * next + block_of<SG>(g, u), nb - 1) * 16));
                if (u == 0) {
                    in.s[t] = run_scales<GSH, SG>(w.s[t], w.vs[t], gs, next, g);
                    if constexpr (MINS) in.m[t] = run_scales<GSH, SG>(w.m[t], w.vs[t], gs, next, g);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            const uint8_t * ap = lds + (active ? (R * 4 + u * 2) * L.step + row * 64 + (SG == 0 ? g * 16 : 0) : L.zero), * ah = ap + (active ? L.step : 0);
            const int at = ((8 * R + block_of<SG>(g, u)) >> SG) * tp + first;
#pragma unroll
            for (int q = 0; q < TM / TG; q++) {
                if (q * TG >= nt) continue;
                const int o = q * TG * P * 64 + (SG == 0 ? 0 : turn<SG>(TG * P % 16 ? row + q * TG * P : row, g) * 16);
                const i32x4 a0 = *reinterpret_cast<const i32x4 *>(ap + o), a1 = *reinterpret_cast<const i32x4 *>(ah + o);
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
                        else if constexpr (P == 2) v = (float) ((c[t][2 * i] << 8) + c[t][2 * i + 1]);
                        else v = __builtin_fmaf((float) ((c[t][0] << 8) + c[t][1]), 256.f, (float) c[t][2]);
                        float & s = acc[t][q * TL + i];
                        s = __builtin_fmaf(v, sc[t][u] * d, s);
                        if constexpr (MINS) s = __builtin_fmaf(mn[t][u], ds[at + q * TG + i], s);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
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

// The slot-th expert that occurs and the pairs that chose it (in any order: a pair's results do not depend on its place); -1 past the last
// one.  Choices that are no expert are left out.
struct Found {
    unsigned mark[ROUTE_MAX_EXPERTS / 32];
    int count;
    uint16_t pairs[MAX_PAIRS];
};
constexpr int FOUND = (sizeof(Found) + 255) & ~255; // its place in LDS, in front of a pass's
__device__ __forceinline__ int find(const int * ids, int pairs, int n_experts, int slot, Found & f) {
    const int lane = threadIdx.x & 63;
    if (pairs <= 64) { // every wave by itself, in the order of their first pairs (the waves write the same list)
        const int id = lane < pairs ? ids[lane] : -1;
        uint64_t todo = __ballot((unsigned) id < (unsigned) n_experts), of = 0;
        int e = -1;
        for (; todo && slot >= 0; slot--) {
            e = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
            of = __ballot(id == e);
            todo &= ~of;
        }
        if (slot >= 0) return -1;
        if (id == e) f.pairs[__builtin_amdgcn_mbcnt_hi((unsigned) (of >> 32), __builtin_amdgcn_mbcnt_lo((unsigned) of, 0))] = (uint16_t) lane;
        f.count = __builtin_popcountll(of);
        __syncthreads();
        return e;
    }
    constexpr int NP = (MAX_PAIRS + WAVES * 64 - 1) / (WAVES * 64);
    int id[NP];
    if (threadIdx.x < ROUTE_MAX_EXPERTS / 32) f.mark[threadIdx.x] = 0;
    if (threadIdx.x == 0) f.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NP; i++) {
        const int p = threadIdx.x + i * WAVES * 64;
        id[i] = p < pairs ? ids[p] : -1;
        if ((unsigned) id[i] < (unsigned) n_experts) atomicOr(&f.mark[id[i] >> 5], 1u << (id[i] & 31));
    }
    __syncthreads();
    unsigned word = lane < 32 ? f.mark[lane] : 0;
    int before = __popc(word);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up(before, d);
        if (lane >= d) before += v;
    }
    before -= __popc(word);
    const uint64_t at = __ballot(before <= slot && slot < before + __popc(word));
    if (!at) return -1;
    const int l = __builtin_ctzll(at);
    word = __builtin_amdgcn_readlane(word, l);
    for (int i = slot - __builtin_amdgcn_readlane(before, l); i > 0; i--) word &= word - 1;
    const int e = l * 32 + __builtin_ctz(word);
#pragma unroll
    for (int i = 0; i < NP; i++)
        if (id[i] == e) f.pairs[atomicAdd(&f.count, 1)] = (uint16_t) (threadIdx.x + i * WAVES * 64);
    __syncthreads();
    return e;
}

__device__ __forceinline__ unsigned lds_address(const uint8_t * lds) {
    return (unsigned) __builtin_amdgcn_readfirstlane((unsigned) (size_t) (const __attribute__((address_space(3))) uint8_t *) lds);
}

// x of nt tokens into LDS
template <int XF, int SG, bool MINS> __device__ __forceinline__ void stage_x(const MoeArgs & a, uint8_t * lds, const Lds & L, int tp, int nt, const uint16_t * pairs) {
    constexpr int P = planes_of(XF);
    const int nb = a.dim >> 5, nbp = padded(nb), tid = threadIdx.x;
    float * dx = reinterpret_cast<float *>(lds + L.dx), * ds = reinterpret_cast<float *>(lds + L.ds);
    if constexpr (XF == W4_UNITS) {
        static_assert(SG == 0, "a unit's blocks have scales of their own");
        const unsigned base = lds_address(lds);
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
        for (int c = wave; c < nbp >> 1; c += WAVES) // a piece of 16 rows a copy
            for (int t0 = 0; t0 < nt; t0 += 16) {
                const int t = t0 + (lane >> 2), g = lane & 3, row = pairs[min(t, nt - 1)] / a.top_k;
                const int block = min((c >> 2) * 8 + block_of<0>(g, c >> 1 & 1), nb - 1);
                const int8_t * from = (block & 1 ? a.xb : a.xa) + ((size_t) row * nb + (block & ~1) + (c & 1)) * 16;
                if (t < nt) dma16(from, base + c * L.step + t0 * 64);
            }
        for (int i = tid; i < nt * nbp; i += WAVES * 64) {
            const int t = i / nbp, block = i - t * nbp, row = pairs[t] / a.top_k;
            float d = 0.f, s = 0.f;
            if (block < nb) {
                const uint16_t * m = a.xmeta + ((size_t) row * nb + (block & ~1)) * 4;
                d = h2f_bits(m[block & 1]);
                if (MINS) s = d * (float) ((int) (int16_t) m[2 + (block & 1)] + (int) (int16_t) m[6 + (block & 1)]);
            }
            dx[block * tp + t] = d * 0.0625f;
            if (MINS) ds[block * tp + t] = s;
        }
        vm_drain();
    } else {
        for (int i = tid; i < nt * nbp * 4; i += WAVES * 64) { // a quarter of a block (4 << SG lanes an exponent)
            const int t = i / (nbp * 4), j = i - t * nbp * 4, block = j >> 2, qt = j & 3;
            float v[8], s = 0.f;
            typename Elem<XF>::Raw8 raw{};
            if (block < nb) raw = Elem<XF>::raw8(static_cast<const typename Elem<XF>::T *>(a.x) + (pairs[t] / a.top_k) * a.x_stride + 32 * block + 8 * qt);
            unsigned top = Elem<XF>::top8(raw);
#pragma unroll
            for (int m = 1; m < 4 << SG; m <<= 1) top = max(top, shfl_xor_u(top, m));
            Elem<XF>::open8(raw, v);
            if (MINS) {
#pragma unroll
                for (int k = 0; k < 8; k++) s += v[k];
#pragma unroll
                for (int m = 1; m < 4 << SG; m <<= 1) s += shfl_xor(s, m);
            }
            const Fixed f = fixed_of<P>(top);
            unsigned out[P][2] = {};
#pragma unroll
            for (int k = 0; k < 8; k++) {
                int q[P];
                planes_split<P>(to_fixed<P>(v[k], f.up), q);
#pragma unroll
                for (int p = 0; p < P; p++) out[p][k >> 2] |= (unsigned) (q[p] & 255) << 8 * (k & 3);
            }
            uint8_t * to = lds + piece_of<SG>(block, qt >> 1) * L.step + 8 * (qt & 1);
#pragma unroll
            for (int p = 0; p < P; p++) *reinterpret_cast<uint2 *>(to + place<SG>(t * P + p, group_in<SG>(block))) = make_uint2(out[p][0], out[p][1]);
            if ((j & ((4 << SG) - 1)) == 0) {
                dx[(block >> SG) * tp + t] = block < nb ? f.dx : 0.f;
                if (MINS) ds[(block >> SG) * tp + t] = s;
            }
        }
    }
}

// the inner values' planes of nt pairs into LDS
template <int P, int SG, bool MINS> __device__ __forceinline__ void stage_h(const MoeArgs & a, uint8_t * lds, const Lds & L, int tp, int nt, const uint16_t * pairs) {
    const int nb = a.inner >> 5, nbp = padded(nb), tid = threadIdx.x, ng = (nb + (1 << SG) - 1) >> SG;
    const unsigned base = lds_address(lds);
    float * dx = reinterpret_cast<float *>(lds + L.dx), * ds = reinterpret_cast<float *>(lds + L.ds);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    for (int c = wave; c < nbp >> 1; c += WAVES) // a piece of 16 rows a copy
        for (int r0 = 0; r0 < nt * P; r0 += 16) {
            const int r = r0 + (lane >> 2), t = min(r / P, nt - 1), g = turn<SG>(r, lane & 3); // (its own inverse)
            if (r < nt * P) dma16(a.hq + ((size_t) pairs[t] * P + (r - t * P)) * nbp * 32 + c * 64 + g * 16, base + c * L.step + r0 * 64);
        }
    for (int i = tid; i < nt * (nbp >> SG); i += WAVES * 64) {
        const int t = i / (nbp >> SG), k = i - t * (nbp >> SG);
        dx[k * tp + t] = k < ng ? a.hd[(size_t) pairs[t] * ng + k] : 0.f;
        if (MINS) ds[k * tp + t] = k < ng ? a.hs[(size_t) pairs[t] * ng + k] : 0.f;
    }
    vm_drain();
}
__device__ __forceinline__ void zero_pieces(uint8_t * lds, const Lds & L) {
    for (int i = threadIdx.x; i < (L.dx - L.zero) / 4; i += WAVES * 64) reinterpret_cast<unsigned *>(lds + L.zero)[i] = 0;
}

// The gate and the up projection: a workgroup has 16 CG inner columns of an expert, its waves (16 columns of both, a KS-th of dim), CG KS = 8.
// SG: lane groups that share a sum of x; SH: those of the down projection, whose x (h) this kernel leaves as planes.
template <int XF, int GSH, int SH, int TM, bool MINS> __global__ __launch_bounds__(WAVES * 64, 4) void k_moe_up(MoeArgs a) {
    constexpr int P = planes_of(XF), HP = inner_planes(XF), SG = P == 1 ? 0 : GSH;
    extern __shared__ __attribute__((aligned(16))) uint8_t all[];
    Found & found = *reinterpret_cast<Found *>(all);
    uint8_t * lds = all + FOUND;
    const int nb = a.dim >> 5, nbp = padded(nb), runs = nbp >> 3, tp = a.tp_up;
    const Lds L = lds_of(P, SG, nbp, tp, MINS);
    float * red = reinterpret_cast<float *>(lds + ((L.end + 15) & ~15)); // [KS][CG][2][tp][16]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int KS = 1 << a.ks_up, CG = WAVES >> a.ks_up, cg = wave & (CG - 1), ks = wave / CG;
    const int e = find(a.ids, a.rows * a.top_k, a.n_experts, blockIdx.y, found);
    if (e < 0) return;
    const int cnt = found.count, gs = (nb + (1 << GSH) - 1) >> GSH, c0 = blockIdx.x * 16 * CG, r0 = (runs * ks) >> a.ks_up, r1 = (runs * (ks + 1)) >> a.ks_up;
    Rows<2> w; // (columns past the last one: zeros below)
    w.set(0, a.up, 2 * e, a.inner, c0 + cg * 16, nb, gs);
    w.set(1, a.up, 2 * e + 1, a.inner, c0 + cg * 16, nb, gs);
    zero_pieces(lds, L);
    for (int t0 = 0; t0 < cnt; t0 += tp) {
        const int nt = min(tp, cnt - t0);
        const Run<2, MINS> first = load_run<GSH, SG, 2, MINS>(w, nb, min(r0, runs - 1)); // (on its way while x is made ready)
        if (t0) __syncthreads();
        stage_x<XF, SG, MINS>(a, lds, L, tp, nt, found.pairs + t0);
        __syncthreads();
        float acc[2][TM >> SG];
        products<P, GSH, SG, 2, TM, MINS>(w, first, nb, r0, r1, lds, L, tp, nt, acc);
        sums_out<P, SG, 2, TM>(acc, tp, nt, red + (ks * CG + cg) * 2 * tp * 16);
        __syncthreads();
        // four columns of a token a thread, 8 << SH threads for the values of an exponent of h
        for (int j = threadIdx.x; j < nt * CG * 4; j += WAVES * 64) {
            const int i = j / (CG * 4), col = (j - i * (CG * 4)) * 4, c = c0 + col;
            f32x4 gt = {0.f, 0.f, 0.f, 0.f}, up = gt, h;
            for (int k = 0; k < KS; k++) {
                const float * p = red + (((k * CG + (col >> 4)) * 2 * tp + i) * 16 + (col & 15));
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
            const Fixed f = fixed_of<HP>(top);
            unsigned out[HP] = {};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                int q[HP];
                planes_split<HP>(to_fixed<HP>(h[k], f.up), q);
#pragma unroll
                for (int p = 0; p < HP; p++) out[p] |= (unsigned) (q[p] & 255) << 8 * k;
            }
            const int nbi = a.inner >> 5, ng = (nbi + (1 << SH) - 1) >> SH, block = c >> 5, pair = found.pairs[t0 + i];
            if (block >= ng << SH) continue; // (what fills the last exponent's values up: zeros)
            uint8_t * to = a.hq + (size_t) pair * HP * padded(nbi) * 32 + piece_of<SH>(block, c >> 4 & 1) * 64 + group_in<SH>(block) * 16 + (c & 15);
#pragma unroll
            for (int p = 0; p < HP; p++) *reinterpret_cast<unsigned *>(to + (size_t) p * padded(nbi) * 32) = out[p];
            if ((c & ((32 << SH) - 1)) == 0) {
                a.hd[(size_t) pair * ng + (block >> SH)] = f.dx;
                if (MINS) a.hs[(size_t) pair * ng + (block >> SH)] = s;
            }
        }
    }
}

// the down projection of every pair: waves (32 columns, a KS-th of inner)
template <int P, int GSH, int SG, int TM, bool MINS> __global__ __launch_bounds__(WAVES * 64, 4) void k_moe_down(MoeArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t all[];
    Found & found = *reinterpret_cast<Found *>(all);
    uint8_t * lds = all + FOUND;
    const int nb = a.inner >> 5, nbp = padded(nb), runs = nbp >> 3, tp = a.tp_down;
    const Lds L = lds_of(P, SG, nbp, tp, MINS);
    float * red = reinterpret_cast<float *>(lds + ((L.end + 15) & ~15)); // [KS][CG][2][tp][16]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int KS = 1 << a.ks_down, CG = WAVES >> a.ks_down, cg = wave & (CG - 1), ks = wave / CG;
    const int e = find(a.ids, a.rows * a.top_k, a.n_experts, blockIdx.y, found);
    if (e < 0) return;
    const int cnt = found.count, gs = (nb + (1 << GSH) - 1) >> GSH, c0 = blockIdx.x * CG * 32, r0 = (runs * ks) >> a.ks_down, r1 = (runs * (ks + 1)) >> a.ks_down;
    Rows<2> w; // (columns past the last one: not stored)
    w.set(0, a.down, e, a.dim, c0 + cg * 32, nb, gs);
    w.set(1, a.down, e, a.dim, c0 + cg * 32 + 16, nb, gs);
    zero_pieces(lds, L);
    for (int t0 = 0; t0 < cnt; t0 += tp) {
        const int nt = min(tp, cnt - t0);
        const Run<2, MINS> first = load_run<GSH, SG, 2, MINS>(w, nb, min(r0, runs - 1));
        if (t0) __syncthreads();
        stage_h<P, SG, MINS>(a, lds, L, tp, nt, found.pairs + t0);
        __syncthreads();
        float acc[2][TM >> SG];
        products<P, GSH, SG, 2, TM, MINS>(w, first, nb, r0, r1, lds, L, tp, nt, acc);
        sums_out<P, SG, 2, TM>(acc, tp, nt, red + (ks * CG + cg) * 2 * tp * 16);
        __syncthreads();
        for (int j = threadIdx.x; j < nt * CG * 8; j += WAVES * 64) {
            const int i = j / (CG * 8), col = (j - i * (CG * 8)) * 4, c = c0 + col;
            if (c >= a.dim) continue;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < KS; k++) v += *reinterpret_cast<const f32x4 *>(red + (((k * CG + (col >> 5)) * 2 + (col >> 4 & 1)) * tp + i) * 16 + (col & 15));
            *reinterpret_cast<f32x4 *>(a.out + (size_t) found.pairs[t0 + i] * a.dim + c) = v;
        }
    }
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

// (the gate's and) a projection's LDS
template <class A> size_t lds_bytes(const A & a, int P, int sg, int blocks, int tp) {
    return FOUND + ((lds_of(P, sg, padded(blocks), tp, a.up.mins).end + 15) & ~15) + (size_t) WAVES * 2 * tp * 16 * 4;
}
template <int XF, int GSH, int SH, int TM, bool MINS> hipError_t up(const MoeArgs & a, int slots, hipStream_t st) {
    constexpr int P = planes_of(XF), SG = P == 1 ? 0 : GSH;
    static std::atomic<uint64_t> done;
    const size_t lds = lds_bytes(a, P, SG, a.dim / 32, a.tp_up);
    const hipError_t e = allow_lds(k_moe_up<XF, GSH, SH, TM, MINS>, lds, done);
    const int cols = 16 * (WAVES >> a.ks_up);
    return e != hipSuccess ? e : launch(k_moe_up<XF, GSH, SH, TM, MINS>, dim3((a.inner + cols - 1) / cols, slots), dim3(WAVES * 64), lds, st, a);
}
template <int P, int GSH, int SG, int TM, bool MINS> hipError_t down(const MoeArgs & a, int slots, hipStream_t st) {
    static std::atomic<uint64_t> done;
    const size_t lds = lds_bytes(a, P, SG, a.inner / 32, a.tp_down);
    const hipError_t e = allow_lds(k_moe_down<P, GSH, SG, TM, MINS>, lds, done);
    const int cols = 32 * (WAVES >> a.ks_down);
    return e != hipSuccess ? e : launch(k_moe_down<P, GSH, SG, TM, MINS>, dim3((a.dim + cols - 1) / cols, slots), dim3(WAVES * 64), lds, st, a);
}
template <int XF, int GSH, int SH, bool MINS> hipError_t run(const MoeArgs & a, hipStream_t st) {
    constexpr int HP = inner_planes(XF), YT = XF == W4_UNITS ? DT_F32 : XF;
    const int slots = std::min(a.n_experts, a.rows * a.top_k);
    hipError_t e = a.tp_up <= 8 ? up<XF, GSH, SH, 8, MINS>(a, slots, st) : up<XF, GSH, SH, 16, MINS>(a, slots, st);
    if (e != hipSuccess) return e;
    e = a.tp_down <= 8 ? down<HP, GSH, SH, 8, MINS>(a, slots, st) : down<HP, GSH, SH, 16, MINS>(a, slots, st);
    if (e != hipSuccess) return e;
    return launch(k_moe_sum<YT>, dim3((a.dim + 1023) / 1024, a.rows), dim3(256), 0, st, a);
}
template <int XF, int GSH, bool MINS> hipError_t run(const MoeArgs & a, hipStream_t st) {
    if constexpr (GSH == 0) return run<XF, 0, 0, MINS>(a, st);
    else return a.ks_up == 0 ? run<XF, GSH, GSH, MINS>(a, st) : run<XF, GSH, 0, MINS>(a, st);
}
template <int XF, bool MINS> hipError_t run(const MoeArgs & a, hipStream_t st) {
    return a.gsh == 0 ? run<XF, 0, MINS>(a, st) : a.gsh == 1 ? run<XF, 1, MINS>(a, st) : run<XF, 2, MINS>(a, st);
}
template <int XF> hipError_t run(const MoeArgs & a, hipStream_t st) { return a.up.mins ? run<XF, true>(a, st) : run<XF, false>(a, st); }

// tokens of a pass: twice what an expert has on average (at most 16), in half of a CU's LDS where that holds an instruction's
int pass_tokens(const MoeArgs & a, int P, int sg, int blocks) {
    const int tg = group_of(P, sg), avg = (a.rows * a.top_k + a.n_experts - 1) / a.n_experts;
    int tp = std::min((std::min(a.rows, std::max(2 * avg, 4)) + tg - 1) / tg * tg, 16);
    while (tp > tg && lds_bytes(a, P, sg, blocks, tp) > 80 * 1024) tp -= tg;
    return tp;
}
// waves that split k: as few as leave `most` workgroups of `cols` columns each (times the waves that share them)
int split(int experts, int n, int cols, int runs, int limit) {
    int log = 0;
    while (log < limit && experts * ((n + (cols * WAVES >> log) - 1) / (cols * WAVES >> log)) < 512 && runs >= 2 << log) log++;
    return log;
}

} // namespace

long long moe_plan(MoeArgs & a, int xform, uint8_t * ws) {
    const int HP = inner_planes(xform), nbi = a.inner / 32;
    const long long pairs = (long long) std::min(a.rows, MOE_ROWS) * a.top_k;
    long long at = 0;
    const auto take = [&](long long bytes) {
        uint8_t * p = ws + at;
        at += (bytes + 255) & ~255ll;
        return p;
    };
    a.hq = take(pairs * HP * padded(nbi) * 32);
    a.hd = reinterpret_cast<float *>(take(pairs * nbi * 4));
    a.hs = reinterpret_cast<float *>(take(a.up.mins ? pairs * nbi * 4 : 0));
    a.out = reinterpret_cast<float *>(take(pairs * a.dim * 4));
    return at;
}

// (of one run of at most MOE_ROWS rows)
static void split_work(MoeArgs & a, int xform) {
    const int HP = inner_planes(xform), P = planes_of(xform), nbi = a.inner / 32;
    const int experts = std::min(a.n_experts, a.rows * a.top_k);
    a.ks_up = split(experts, a.inner, 16, padded(a.dim / 32) / 8, 2);
    a.ks_down = split(experts, a.dim, 32, padded(nbi) / 8, 3);
    a.tp_up = pass_tokens(a, P, P == 1 ? 0 : a.gsh, a.dim / 32);
    a.tp_down = pass_tokens(a, HP, a.ks_up == 0 ? a.gsh : 0, nbi);
}

hipError_t launch_moe(const MoeArgs & all, int xform, hipStream_t st) {
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
        const hipError_t e = xform == W4_UNITS ? run<W4_UNITS>(a, st) : xform == DT_F32 ? run<DT_F32>(a, st) : xform == DT_F16 ? run<DT_F16>(a, st) : run<DT_BF16>(a, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

} // namespace qkv
