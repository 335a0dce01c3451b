// A mixture-of-experts layer with 4-bit weights for a few tokens: h = silu(G x) (U x) of every (token, expert) pair, then
// y[m] = sum over the row's experts of w D h.  Three kernels: the gate's and the up projection's rows together, the down projection of every
// pair, and the sum over a row's experts in their order (no atomics: the same bits every time).
//
// Workgroups stand for (a tile of weight rows, one of the experts that occur); each finds its expert and the pairs that chose it in
// the row's choices itself.  An expert has few tokens, so what counts is the way of its codes: from HBM, and from 4 bits to an operand.  Codes
// become int8 with four vector instructions for 8 of them (fp16 takes 13), so x is made integer too: per block of 32 values an exponent,
// and two or three int8 planes (14 bits of the block's largest power of two for 16-bit x, 22 for fp32; int8 units are one plane as they are).  The
// matrix instruction's sums are exact, a block's scales multiply its sum in fp32.
//
// A wave has two tiles of 16 weight rows.  Lane (n = lane & 15, g = lane >> 4) loads the 16 bytes of block 8 R + 2 g + u of row n, u = 0, 1:
// 32 bytes of its own, the 128 of a cache line for a row's four lanes, and both scales in 4 bytes.  The instruction contracts over all four
// lane groups, but every block has scales of its own, so the planes go in on the diagonal: operand row 4 b + m holds plane m of block
// b in lane group b and zeros in the others, and output row 4 b + m is that block's sum, in the lanes that hold its scale.
#include "step_dev.h"
#include "step_mix_launch.h"

#include <algorithm>

namespace qkv {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32_u2 __attribute__((aligned(2)));

constexpr int T_MAX = 16;     // tokens of an expert in a pass
constexpr int MAX_PAIRS = MOE_ROWS * ROUTE_MAX_TOP;
constexpr int WAVES = 8;

constexpr int planes_of(int xform) { return xform == W4_UNITS ? 1 : xform == DT_F32 ? 3 : 2; }
constexpr int inner_planes(int xform) { return xform == DT_F16 || xform == DT_BF16 ? 2 : 3; } // (y is fp32 else)
constexpr int group_of(int P) { return P == 1 ? 4 : P == 2 ? 2 : 1; } // tokens of one matrix instruction

// LDS of a pass: rows of planes (token t's plane p is row t P + p), each [runs of 8 blocks][u][half][g][16 bytes], the rows 64 bytes
// past a multiple of 256 so that an instruction's 16 pieces lie in different banks; 128 zeros; per block the tokens' factors, and
// with minimums the tokens' sums
struct Lds {
    int row, zero, dx, ds, end;
};
__host__ __device__ __forceinline__ constexpr Lds lds_of(int P, int nbp, int tp, bool mins) {
    Lds l{};
    l.row = nbp * 32 + 64;
    l.zero = tp * P * l.row;
    l.dx = l.zero + 128;
    l.ds = l.dx + nbp * tp * 4;
    l.end = mins ? l.ds + nbp * tp * 4 : l.ds;
    return l;
}
__host__ __device__ __forceinline__ constexpr int padded(int blocks) { return (blocks + 7) & ~7; }
// the place in a row of 16 bytes of a block
__device__ __forceinline__ int piece(int block, int half) { return ((block >> 3) * 4 + (block & 1) * 2 + half) * 64 + (block >> 1 & 3) * 16; }

// a block's values as integers: times `up`, a power of two that brings the largest to [2^13, 2^14) (three planes: [2^21, 2^22)), and the
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

// two tiles of 16 weight rows, the lane's row of each
struct Rows {
    const uint8_t * c[2];
    const uint16_t * s[2], * m[2];
};
// the sums of runs r0 .. r1 - 1 (of 8 blocks) for nt tokens in LDS
template <int P, int GSH, bool MINS>
__device__ __forceinline__ void products(const Rows & w, int nb, int r0, int r1, const uint8_t * lds, const Lds & L, int tp, int nt, float (&acc)[2][T_MAX]) {
    constexpr int TG = group_of(P), VR = TG * P; // tokens and operand rows of an instruction
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, m = n & 3, gs = (nb + (1 << GSH) - 1) >> GSH;
    const bool active = n >> 2 == g && m < VR;
    const int aoff = active ? m * L.row + g * 16 : L.zero;
    const unsigned amask = active ? ~0u : 0u;
    const float * dx = reinterpret_cast<const float *>(lds + L.dx), * ds = reinterpret_cast<const float *>(lds + L.ds);
    struct Run {
        u32x4 c[2][2];
        unsigned s[2], m[2]; // two scales
    };
    const auto scales = [&](const uint16_t * p, int R) -> unsigned {
        if constexpr (GSH == 0) {
            if (8 * R + 8 <= nb) return *reinterpret_cast<const u32_u2 *>(p + 8 * R + 2 * g);
            return p[min(8 * R + 2 * g, nb - 1)] | (unsigned) p[min(8 * R + 2 * g + 1, nb - 1)] << 16;
        } else return p[min((8 * R + 2 * g) >> GSH, gs - 1)];
    };
    const auto load = [&](int R) {
        Run r;
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int u = 0; u < 2; u++) r.c[t][u] = *reinterpret_cast<const u32x4 *>(w.c[t] + min(8 * R + 2 * g + u, nb - 1) * 16); // (past the last block factors of zero)
            r.s[t] = scales(w.s[t], R);
            if constexpr (MINS) r.m[t] = scales(w.m[t], R);
        }
        return r;
    };
    if (r0 >= r1) return;
    Run nx = load(r0);
#pragma unroll 1
    for (int R = r0; R < r1; R++) {
        const Run cu = nx;
        if (R + 1 < r1) nx = load(R + 1);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            i32x4 b[2][2];
            float sc[2], mn[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    int t0, t1;
                    w4_bytes(cu.c[t][u][k], t0, t1);
                    b[t][k >> 1][2 * (k & 1)] = t0;
                    b[t][k >> 1][2 * (k & 1) + 1] = t1;
                }
                sc[t] = h2f_bits((uint16_t) (cu.s[t] >> (GSH == 0 ? 16 * u : 0)));
                if constexpr (MINS) mn[t] = h2f_bits((uint16_t) (cu.m[t] >> (GSH == 0 ? 16 * u : 0)));
            }
            const int block = 8 * R + 2 * g + u;
#pragma unroll
            for (int q = 0; q < T_MAX / TG; q++) {
                if (q * TG >= nt) continue;
                const uint8_t * ap = lds + aoff + ((unsigned) (q * VR * L.row + (R * 4 + u * 2) * 64) & amask);
                const i32x4 a0 = *reinterpret_cast<const i32x4 *>(ap), a1 = *reinterpret_cast<const i32x4 *>(ap + 64);
                i32x4 c[2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    c[t] = i32x4{0, 0, 0, 0};
                    c[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, b[t][0], c[t], 0, 0, 0);
                    c[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, b[t][1], c[t], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < TG; i++) {
                    const float d = dx[block * tp + q * TG + i];
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        float v;
                        if constexpr (P == 1) v = (float) c[t][i];
                        else if constexpr (P == 2) v = (float) ((c[t][2 * i] << 8) + c[t][2 * i + 1]);
                        else v = __builtin_fmaf((float) ((c[t][0] << 8) + c[t][1]), 256.f, (float) c[t][2]);
                        float & s = acc[t][q * TG + i];
                        s = __builtin_fmaf(v, sc[t] * d, s);
                        if constexpr (MINS) s = __builtin_fmaf(mn[t], ds[block * tp + q * TG + i], s);
                    }
                }
            }
        }
    }
}

// The slot-th expert that occurs (ascending) and the pairs that chose it (in any order: a pair's results do not depend on its place);
// -1 past the last one.  Choices that are no expert are left out.
struct Found {
    unsigned mark[ROUTE_MAX_EXPERTS / 32];
    int count;
    uint16_t pairs[MAX_PAIRS];
};
constexpr int FOUND = (sizeof(Found) + 255) & ~255; // its place in LDS, in front of a pass's
__device__ __forceinline__ int find(const int * ids, int pairs, int n_experts, int slot, Found & f) {
    constexpr int NP = (MAX_PAIRS + WAVES * 64 - 1) / (WAVES * 64);
    const int lane = threadIdx.x & 63;
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

// x of tokens t0 .. t0 + nt - 1 of the expert into LDS
template <int XF, bool MINS> __device__ __forceinline__ void stage_x(const MoeArgs & a, uint8_t * lds, const Lds & L, int tp, int nt, const uint16_t * pairs) {
    constexpr int P = planes_of(XF);
    const int nb = a.dim >> 5, nbp = padded(nb), tid = threadIdx.x;
    float * dx = reinterpret_cast<float *>(lds + L.dx), * ds = reinterpret_cast<float *>(lds + L.ds);
    if constexpr (XF == W4_UNITS) {
        const unsigned base = lds_address(lds);
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, per = (nbp * 2 + 63) >> 6;
        for (int c = wave; c < nt * per; c += WAVES) { // 64 pieces a copy
            const int t = c / per, i = (c - t * per) * 64 + lane, row = pairs[t] / a.top_k;
            const int block = min((i >> 4) * 8 + (i & 3) * 2 + (i >> 3 & 1), nb - 1);
            const int8_t * from = (block & 1 ? a.xb : a.xa) + ((size_t) row * nb + (block & ~1) + (i >> 2 & 1)) * 16;
            if (i < nbp * 2) dma16(from, base + t * L.row + (c - t * per) * 1024);
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
        for (int i = tid; i < nt * nbp * 4; i += WAVES * 64) { // a quarter of a block
            const int t = i / (nbp * 4), j = i - t * nbp * 4, block = j >> 2, qt = j & 3;
            const bool in = block < nb;
            float v[8], s = 0.f;
            typename Elem<XF>::Raw8 raw{};
            if (in) raw = Elem<XF>::raw8(static_cast<const typename Elem<XF>::T *>(a.x) + (pairs[t] / a.top_k) * a.x_stride + 32 * block + 8 * qt);
            unsigned top = Elem<XF>::top8(raw);
            top = max(top, shfl_xor_u(top, 1));
            top = max(top, shfl_xor_u(top, 2));
            Elem<XF>::open8(raw, v);
            if (MINS) {
#pragma unroll
                for (int k = 0; k < 8; k++) s += v[k];
                s += shfl_xor(s, 1);
                s += shfl_xor(s, 2);
            }
            const Fixed f = fixed_of<P>(top);
            unsigned out[P][2] = {};
#pragma unroll
            for (int k = 0; k < 8; k++) {
                int q[P];
                planes_split<P>((int) __builtin_rintf(v[k] * f.up), q);
#pragma unroll
                for (int p = 0; p < P; p++) out[p][k >> 2] |= (unsigned) (q[p] & 255) << 8 * (k & 3);
            }
            uint8_t * to = lds + t * P * L.row + piece(block, qt >> 1) + 8 * (qt & 1);
#pragma unroll
            for (int p = 0; p < P; p++) *reinterpret_cast<uint2 *>(to + p * L.row) = make_uint2(out[p][0], out[p][1]);
            if (qt == 0) {
                dx[block * tp + t] = in ? f.dx : 0.f;
                if (MINS) ds[block * tp + t] = s;
            }
        }
    }
}

// the inner values' planes of an expert's tokens into LDS
template <int P, bool MINS> __device__ __forceinline__ void stage_h(const MoeArgs & a, uint8_t * lds, const Lds & L, int tp, int nt, const uint16_t * pairs) {
    const int nb = a.inner >> 5, nbp = padded(nb), tid = threadIdx.x, per = (nbp * 2 + 63) >> 6;
    const unsigned base = lds_address(lds);
    float * dx = reinterpret_cast<float *>(lds + L.dx), * ds = reinterpret_cast<float *>(lds + L.ds);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    for (int c = wave; c < nt * P * per; c += WAVES) {
        const int r = c / per, t = r / P, i = (c - r * per) * 64 + lane;
        if (i < nbp * 2) dma16(a.hq + ((size_t) pairs[t] * P + (r - t * P)) * nbp * 32 + i * 16, base + r * L.row + (c - r * per) * 1024);
    }
    for (int i = tid; i < nt * nbp; i += WAVES * 64) {
        const int t = i / nbp, block = i - t * nbp;
        dx[block * tp + t] = block < nb ? a.hd[(size_t) pairs[t] * nb + block] : 0.f;
        if (MINS) ds[block * tp + t] = block < nb ? a.hs[(size_t) pairs[t] * nb + block] : 0.f;
    }
    vm_drain();
}
__device__ __forceinline__ void zero_pieces(uint8_t * lds, const Lds & L) {
    if (threadIdx.x < 32) reinterpret_cast<unsigned *>(lds + L.zero)[threadIdx.x] = 0;
}

// h of 32 inner columns for the expert's tokens: waves (half of the columns, a quarter of dim)
template <int XF, int GSH, bool MINS> __global__ __launch_bounds__(WAVES * 64, 2) void k_moe_up(MoeArgs a) {
    constexpr int P = planes_of(XF), HP = inner_planes(XF), KS = WAVES / 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t all[];
    Found & found = *reinterpret_cast<Found *>(all);
    uint8_t * lds = all + FOUND;
    const int nb = a.dim >> 5, nbp = padded(nb), runs = nbp >> 3, tp = a.tp_up;
    const Lds L = lds_of(P, nbp, tp, MINS);
    float * red = reinterpret_cast<float *>(lds + ((L.end + 15) & ~15)); // [KS][2 halves][2][tp][16]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, half = wave & 1, ks = wave >> 1;
    const int e = find(a.ids, a.rows * a.top_k, a.n_experts, blockIdx.y, found);
    if (e < 0) return;
    const int cnt = found.count, gs = (nb + (1 << GSH) - 1) >> GSH;
    Rows w;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const size_t r = (size_t) e * 2 * a.inner + t * a.inner + blockIdx.x * 32 + half * 16 + n;
        w.c[t] = a.up.codes + r * (a.dim >> 1);
        w.s[t] = a.up.scales + r * gs;
        w.m[t] = MINS ? a.up.mins + r * gs : nullptr;
    }
    zero_pieces(lds, L);
    for (int t0 = 0; t0 < cnt; t0 += tp) {
        const int nt = min(tp, cnt - t0);
        if (t0) __syncthreads();
        stage_x<XF, MINS>(a, lds, L, tp, nt, found.pairs + t0);
        __syncthreads();
        float acc[2][T_MAX];
#pragma unroll
        for (int i = 0; i < T_MAX; i++) acc[0][i] = acc[1][i] = 0.f;
        products<P, GSH, MINS>(w, nb, runs * ks / KS, runs * (ks + 1) / KS, lds, L, tp, nt, acc);
#pragma unroll
        for (int i = 0; i < T_MAX; i++) {
            if (i >= nt) continue;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const float v = quad_sum(acc[t][i]);
                if (lane < 16) red[(((ks * 2 + half) * 2 + t) * tp + i) * 16 + n] = v;
            }
        }
        __syncthreads();
        // 32 lanes per token: its 32 columns, one block of the down projection's x
        const int i = threadIdx.x >> 5, col = threadIdx.x & 31;
        if (i < nt) {
            float gt = 0.f, up = 0.f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const int at = (k * 2 + (col >> 4)) * 2;
                gt += red[(at * tp + i) * 16 + (col & 15)];
                up += red[((at + 1) * tp + i) * 16 + (col & 15)];
            }
            const float h = gt / (1.f + expf(-gt)) * up;
            unsigned top = __builtin_bit_cast(unsigned, h) & 0x7fffffffu;
            float s = h;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                top = max(top, shfl_xor_u(top, m));
                if (MINS) s += shfl_xor(s, m);
            }
            const Fixed f = fixed_of<HP>(top);
            int q[HP];
            planes_split<HP>((int) __builtin_rintf(f.up == 0.f ? 0.f : h * f.up), q);
            const int nbi = a.inner >> 5, block = blockIdx.x, pair = found.pairs[t0 + i];
            uint8_t * to = a.hq + (size_t) pair * HP * padded(nbi) * 32 + piece(block, col >> 4) + (col & 15);
#pragma unroll
            for (int p = 0; p < HP; p++) to[(size_t) p * padded(nbi) * 32] = (uint8_t) q[p];
            if (col == 0) {
                a.hd[(size_t) pair * nbi + block] = f.dx;
                if (MINS) a.hs[(size_t) pair * nbi + block] = s;
            }
        }
    }
}

// the down projection of every pair: waves (32 columns, a part of inner), 1 << ks_log parts
struct DownArgs {
    MoeArgs a;
    int ks_log;
};
template <int P, int GSH, bool MINS> __global__ __launch_bounds__(WAVES * 64, 2) void k_moe_down(DownArgs d) {
    const MoeArgs & a = d.a;
    extern __shared__ __attribute__((aligned(16))) uint8_t all[];
    Found & found = *reinterpret_cast<Found *>(all);
    uint8_t * lds = all + FOUND;
    const int nb = a.inner >> 5, nbp = padded(nb), runs = nbp >> 3, tp = a.tp_down;
    const Lds L = lds_of(P, nbp, tp, MINS);
    float * red = reinterpret_cast<float *>(lds + ((L.end + 15) & ~15)); // [waves][2][tp][16]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15;
    const int KS = 1 << d.ks_log, ks = wave & (KS - 1), cg = wave >> d.ks_log, CG = WAVES >> d.ks_log;
    const int e = find(a.ids, a.rows * a.top_k, a.n_experts, blockIdx.y, found);
    if (e < 0) return;
    const int cnt = found.count, gs = (nb + (1 << GSH) - 1) >> GSH, c0 = blockIdx.x * CG * 32;
    Rows w;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const size_t r = (size_t) e * a.dim + min(c0 + cg * 32 + t * 16 + n, a.dim - 1); // (columns past the last one: not stored)
        w.c[t] = a.down.codes + r * (a.inner >> 1);
        w.s[t] = a.down.scales + r * gs;
        w.m[t] = MINS ? a.down.mins + r * gs : nullptr;
    }
    zero_pieces(lds, L);
    for (int t0 = 0; t0 < cnt; t0 += tp) {
        const int nt = min(tp, cnt - t0);
        if (t0) __syncthreads();
        stage_h<P, MINS>(a, lds, L, tp, nt, found.pairs + t0);
        __syncthreads();
        float acc[2][T_MAX];
#pragma unroll
        for (int i = 0; i < T_MAX; i++) acc[0][i] = acc[1][i] = 0.f;
        products<P, GSH, MINS>(w, nb, (runs * ks) >> d.ks_log, (runs * (ks + 1)) >> d.ks_log, lds, L, tp, nt, acc);
#pragma unroll
        for (int i = 0; i < T_MAX; i++) {
            if (i >= nt) continue;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const float v = quad_sum(acc[t][i]);
                if (lane < 16) red[((wave * 2 + t) * tp + i) * 16 + n] = v;
            }
        }
        __syncthreads();
        for (int j = threadIdx.x; j < nt * CG * 32; j += WAVES * 64) {
            const int i = j / (CG * 32), col = j - i * (CG * 32), c = c0 + col;
            if (c >= a.dim) continue;
            float v = 0.f;
            for (int k = 0; k < KS; k++) v += red[((((col >> 5) * KS + k) * 2 + (col >> 4 & 1)) * tp + i) * 16 + (col & 15)];
            a.out[(size_t) found.pairs[t0 + i] * a.dim + c] = v;
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

template <int XF, int GSH, bool MINS> hipError_t run(const MoeArgs & a, hipStream_t st) {
    constexpr int P = planes_of(XF), HP = inner_planes(XF);
    static std::atomic<uint64_t> done_up, done_down;
    const int slots = std::min(a.n_experts, a.rows * a.top_k);
    size_t lds = FOUND + ((lds_of(P, padded(a.dim / 32), a.tp_up, MINS).end + 15) & ~15) + (size_t) WAVES * 2 * a.tp_up * 16 * 4;
    hipError_t e = allow_lds(k_moe_up<XF, GSH, MINS>, lds, done_up);
    if (e != hipSuccess) return e;
    e = launch(k_moe_up<XF, GSH, MINS>, dim3(a.inner / 32, slots), dim3(WAVES * 64), lds, st, a);
    if (e != hipSuccess) return e;
    const int runs = padded(a.inner / 32) / 8;
    DownArgs d{a, runs >= 4 ? 2 : runs >= 2 ? 1 : 0};
    lds = FOUND + ((lds_of(HP, padded(a.inner / 32), a.tp_down, MINS).end + 15) & ~15) + (size_t) WAVES * 2 * a.tp_down * 16 * 4;
    e = allow_lds(k_moe_down<HP, GSH, MINS>, lds, done_down);
    if (e != hipSuccess) return e;
    const int cols = 32 * (WAVES >> d.ks_log);
    e = launch(k_moe_down<HP, GSH, MINS>, dim3((a.dim + cols - 1) / cols, slots), dim3(WAVES * 64), lds, st, d);
    if (e != hipSuccess) return e;
    constexpr int YT = XF == W4_UNITS ? DT_F32 : XF;
    return launch(k_moe_sum<YT>, dim3((a.dim + 1023) / 1024, a.rows), dim3(256), 0, st, a);
}
template <int XF, bool MINS> hipError_t run(const MoeArgs & a, hipStream_t st) {
    return a.gsh == 0 ? run<XF, 0, MINS>(a, st) : a.gsh == 1 ? run<XF, 1, MINS>(a, st) : run<XF, 2, MINS>(a, st);
}
template <int XF> hipError_t run(const MoeArgs & a, hipStream_t st) { return a.up.mins ? run<XF, true>(a, st) : run<XF, false>(a, st); }

// tokens of a pass: twice what an expert has on average, in at most `most` bytes of LDS, at least one instruction's
int pass_tokens(const MoeArgs & a, int P, int blocks, int most) {
    const int tg = group_of(P), avg = (a.rows * a.top_k + a.n_experts - 1) / a.n_experts;
    int tp = (std::min(a.rows, std::max(2 * avg, 4)) + tg - 1) / tg * tg;
    tp = std::min(tp, T_MAX);
    while (tp > tg && lds_of(P, padded(blocks), tp, a.up.mins).end + WAVES * 2 * tp * 64 + FOUND > most) tp -= tg;
    return tp;
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
    constexpr int HALF = 72 * 1024; // two workgroups per CU
    MoeArgs b = a;
    b.rows = std::min(a.rows, MOE_ROWS);
    a.tp_up = pass_tokens(b, planes_of(xform), a.dim / 32, HALF);
    a.tp_down = pass_tokens(b, HP, nbi, HALF);
    return at;
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
        const hipError_t e = xform == W4_UNITS ? run<W4_UNITS>(a, st) : xform == DT_F32 ? run<DT_F32>(a, st) : xform == DT_F16 ? run<DT_F16>(a, st) : run<DT_BF16>(a, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

} // namespace qkv
