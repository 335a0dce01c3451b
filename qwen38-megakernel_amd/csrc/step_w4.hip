// Products of a few activation rows with 4-bit weights: y[m][j] = sum_k W[j][k] x[m][k], W = s (code - 8) + m with one
// fp16 scale s (and optional fp16 m) per group of 32, 64 or 128 values of a row.  x is either int8 units (codes of 8 bits
// and an fp16 scale per 32 values: what the attention's epilogue and the norm leave) or plain fp32 / fp16 / bf16 rows.
//
// A wave takes 16 weight rows; lane (n = lane & 15, g = lane >> 4) loads 16 bytes, the 32 codes of block 4 s + g of row n,
// per step s.  The matrix instruction contracts over all four lane groups, but every block has scales of its own, so the
// activation operand is laid out on the diagonal: its row 4 b + m holds x[m] of block b in lane group b and zeros in the
// other groups.  Output row 4 b + m is then block b's sum alone, and it lies in the lanes of group b, which hold that
// block's weight scale: one conversion and two products per (row, block) fold it into the row's fp32 sum.  The int8 sums
// are exact; plain rows go in as fp16 with one power of two per (row, block) taken out (fp32 as two such parts).
#include "step_dev.h"

#include <algorithm>

namespace qkv {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int W4_WAVES = 8;
enum { XM_UNITS = 0, XM_HALF = 1, XM_SPLIT = 2 }; // x as int8 units, as one fp16 part, as two

// 16-byte planes per block of 32 values in LDS
constexpr int planes(int mode) { return mode == XM_UNITS ? 2 : mode == XM_HALF ? 4 : 8; }

// LDS: [kcb blocks][planes][MR rows][16 bytes], a zero region of one block's size, then [kcb][MR] float factors of the
// blocks' sums and [kcb][MR] float factors of m
template <int MODE, int MR> __device__ __forceinline__ constexpr int blk_bytes() { return planes(MODE) * MR * 16; }

template <int MODE, int DT, int MR>
__device__ __forceinline__ void w4_stage(const W4Args & a, uint8_t * lds, int row0, int b0, int nblk) {
    constexpr int BB = blk_bytes<MODE, MR>();
    const int nb = a.k >> 5, tid = threadIdx.x;
    float * dx = reinterpret_cast<float *>(lds + (size_t) (a.kcb + 1) * BB), * ds = dx + a.kcb * MR;
    for (int i = tid; i < BB / 16; i += W4_WAVES * 64) reinterpret_cast<uint4 *>(lds + (size_t) a.kcb * BB)[i] = make_uint4(0, 0, 0, 0);
    if constexpr (MODE == XM_UNITS) {
        // (block, half, row) pieces of 16 bytes; the lane of half 0 brings the block's scale and sum
        for (int i = tid; i < nblk * 2 * MR; i += W4_WAVES * 64) {
            const int m = i % MR, half = (i / MR) & 1, bl = i / (2 * MR), blk = b0 + bl, row = row0 + m;
            uint4 v = make_uint4(0, 0, 0, 0);
            float d = 0.f, s = 0.f;
            if (row < a.rows && blk < nb) {
                const int part = blk & 1;
                const size_t gi = (size_t) row * nb + (blk & ~1) + half;
                v = *reinterpret_cast<const uint4 *>((part ? a.xb : a.xa) + gi * 16);
                if (!half) {
                    d = h2f_bits(a.xmeta[gi * 4 + part]);
                    s = d * (float) ((int) (int16_t) a.xmeta[gi * 4 + 2 + part] + (int) (int16_t) a.xmeta[gi * 4 + 6 + part]);
                }
            }
            *reinterpret_cast<uint4 *>(lds + (size_t) bl * BB + (half * MR + m) * 16) = v;
            if (!half) {
                dx[bl * MR + m] = d * 0.0625f; // (the codes go in 16 times as large)
                ds[bl * MR + m] = s;
            }
        }
    } else {
        // a quarter of a block (8 values) per lane
        const typename Elem<DT>::T * x = static_cast<const typename Elem<DT>::T *>(a.x);
        for (int i = tid; i < nblk * 4 * MR; i += W4_WAVES * 64) { // (a multiple of 4 lanes: whole blocks)
            const int q = i & 3, m = (i >> 2) % MR, bl = (i >> 2) / MR, blk = b0 + bl, row = row0 + m;
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (row < a.rows && blk < nb) Elem<DT>::load8(x + (long long) row * a.x_stride + 32 * blk + 8 * q, v);
            float am = 0.f, s = 0.f;
            unsigned top = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                am = fmaxf(am, fabsf(v[k]));
                top = max(top, __builtin_bit_cast(unsigned, v[k]) & 0x7fffffffu);
                s += v[k];
            }
            am = fmaxf(am, shfl_xor(am, 1));
            am = fmaxf(am, shfl_xor(am, 2));
            s += shfl_xor(s, 1);
            s += shfl_xor(s, 2);
            top = max(top, shfl_xor_u(top, 1));
            top = max(top, shfl_xor_u(top, 2));
            // 2^e with the block's largest value in [2^14, 2^15); a block with an infinity or a NaN goes in as it is, its
            // finite values as zeros (they cannot change the result)
            const bool wild = top >= 0x7f800000u;
            const int E = max((int) (top >> 23), 15);
            const float up = wild ? 1.f : __builtin_bit_cast(float, (unsigned) (268 - E) << 23);
            half8 hi, lo;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float t = wild && __builtin_fabsf(v[k]) < __builtin_inff() ? 0.f : v[k] * up;
                const _Float16 h = (_Float16) t;
                // element order of the codes' fp16 pairs: (0, 2) (1, 3) (4, 6) (5, 7)
                const int e = (k & 4) + 2 * (k & 1) + ((k >> 1) & 1);
                hi[e] = h;
                lo[e] = wild ? (_Float16) 0.f : (_Float16) (t - (float) h);
            }
            *reinterpret_cast<half8 *>(lds + (size_t) bl * BB + (q * MR + m) * 16) = hi;
            if constexpr (MODE == XM_SPLIT) *reinterpret_cast<half8 *>(lds + (size_t) bl * BB + ((4 + q) * MR + m) * 16) = lo;
            if (q == 0) {
                dx[bl * MR + m] = wild ? 1.f : __builtin_bit_cast(float, (unsigned) (E - 14) << 23);
                ds[bl * MR + m] = s;
            }
        }
    }
}

// the codes of one word as the four int8 pairs of dwords, 16 (code - 8): values 0..3, values 4..7
__device__ __forceinline__ void w4_bytes(unsigned w, int & lo, int & hi) {
    w ^= 0x88888888u;
    lo = (int) ((w << 4) & 0xf0f0f0f0u);
    hi = (int) (w & 0xf0f0f0f0u);
}
// ... as fp16 pairs (0, 2) (1, 3) (4, 6) (5, 7): 0x6400 | n is 1024 + n exactly
__device__ __forceinline__ half8 w4_halves(unsigned w) {
    const half2v b = {(_Float16) -1032.f, (_Float16) -1032.f};
    const half2v p0 = as_h2((w & 0x000f000fu) | 0x64006400u) + b, p1 = as_h2(((w >> 8) & 0x000f000fu) | 0x64006400u) + b,
                 p2 = as_h2(((w >> 4) & 0x000f000fu) | 0x64006400u) + b, p3 = as_h2(((w >> 12) & 0x000f000fu) | 0x64006400u) + b;
    return half8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// NR activation rows per group of four operand rows (4, or 1 / 2 with one group), RG groups: MR = NR RG rows a pass
template <int MODE, int DT, int NR, int RG>
__global__ __launch_bounds__(W4_WAVES * 64) void k_w4(W4Args a) {
    constexpr int MR = NR * RG, BB = blk_bytes<MODE, MR>();
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const float * dx = reinterpret_cast<const float *>(lds + (size_t) (a.kcb + 1) * BB), * ds = dx + a.kcb * MR;
    float * red = const_cast<float *>(ds) + a.kcb * MR; // [2][waves][MR][16]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int WK = 1 << a.wk_log, wk = wave & (WK - 1), wn = wave >> a.wk_log, WN = W4_WAVES >> a.wk_log;
    const int nb = a.k >> 5, tiles = (a.n + 15) >> 4, sets = (tiles + WN - 1) / WN;
    const int row0 = blockIdx.y * MR;
    // the lane's piece of the diagonal operand: row n = 4 b + m, lane group b
    const int m = n & 3;
    const bool active = (n >> 2) == g && m < NR;
    const int abase = active ? g * BB + m * 16 : a.kcb * BB, astep = active ? 4 * BB : 0;
    const size_t rowb = (size_t) a.k >> 1;
    int par = 0;
    bool staged = false;
    for (int set = blockIdx.x; set < sets; set += gridDim.x, par ^= 1) {
        const int tile = set * WN + wn, row = min(tile * 16 + n, a.n - 1);
        const uint8_t * cp = a.codes + (size_t) row * rowb;
        const size_t sp = (size_t) row * a.gs;
        float acc[RG][NR];
#pragma unroll
        for (int i = 0; i < RG; i++)
#pragma unroll
            for (int r = 0; r < NR; r++) acc[i][r] = 0.f;
        for (int b0 = 0; b0 < nb; b0 += a.kcb) {
            const int nblk = min(a.kcb, (nb - b0 + 3) & ~3);
            if (!staged) {
                __syncthreads();
                w4_stage<MODE, DT, MR>(a, lds, row0, b0, nblk);
                __syncthreads();
                staged = nb <= a.kcb;
            }
            for (int s = wk; s < nblk >> 2; s += WK) {
                const int blk = min(b0 + 4 * s + g, nb - 1); // (past the last block x is zero)
                const u32x4 w = *reinterpret_cast<const u32x4 *>(cp + (size_t) blk * 16);
                const float sc = h2f_bits(a.scales[sp + (blk >> a.gsh)]);
                const uint8_t * ap = lds + abase + s * astep;
                const float * dxp = dx + (4 * s + g) * MR, * dsp = ds + (4 * s + g) * MR;
                const float mn = a.mins ? h2f_bits(a.mins[sp + (blk >> a.gsh)]) : 0.f;
                if constexpr (MODE == XM_UNITS) {
                    i32x4 h0, h1;
                    int t0, t1;
                    w4_bytes(w[0], t0, t1), h0[0] = t0, h0[1] = t1;
                    w4_bytes(w[1], t0, t1), h0[2] = t0, h0[3] = t1;
                    w4_bytes(w[2], t0, t1), h1[0] = t0, h1[1] = t1;
                    w4_bytes(w[3], t0, t1), h1[2] = t0, h1[3] = t1;
#pragma unroll
                    for (int i = 0; i < RG; i++) {
                        const i32x4 a0 = *reinterpret_cast<const i32x4 *>(ap + i * 64), a1 = *reinterpret_cast<const i32x4 *>(ap + MR * 16 + i * 64);
                        i32x4 c = {0, 0, 0, 0};
                        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, h0, c, 0, 0, 0);
                        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, h1, c, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < NR; r++) acc[i][r] = __builtin_fmaf((float) c[r], sc * dxp[4 * i + r], acc[i][r]);
                    }
                } else {
                    half8 hw[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) hw[k] = w4_halves(w[k]);
#pragma unroll
                    for (int i = 0; i < RG; i++) {
                        f32x4 c = {0, 0, 0, 0};
#pragma unroll
                        for (int k = planes(MODE) - 1; k >= 0; k--)
                            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const half8 *>(ap + k * MR * 16 + i * 64), hw[k & 3], c, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < NR; r++) acc[i][r] = __builtin_fmaf(c[r], sc * dxp[4 * i + r], acc[i][r]);
                    }
                }
                if (a.mins) {
#pragma unroll
                    for (int i = 0; i < RG; i++)
#pragma unroll
                        for (int r = 0; r < NR; r++) acc[i][r] = __builtin_fmaf(mn, dsp[4 * i + r], acc[i][r]);
                }
            }
        }
        // the four lane groups' blocks, then the waves of the tile in order
#pragma unroll
        for (int i = 0; i < RG; i++)
#pragma unroll
            for (int r = 0; r < NR; r++) acc[i][r] = quad_sum(acc[i][r]);
        if (WK == 1) {
            if (g == 0 && tile * 16 + n < a.n) {
#pragma unroll
                for (int i = 0; i < MR; i++)
                    if (row0 + i < a.rows) a.y[(long long) (row0 + i) * a.y_stride + tile * 16 + n] = acc[i / NR][i % NR];
            }
            continue;
        }
        float * rp = red + par * (W4_WAVES * MR * 16);
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < MR; i++) rp[(wave * MR + i) * 16 + n] = acc[i / NR][i % NR];
        }
        __syncthreads(); // (the other parity's sums are not written again before every wave has passed this barrier)
        for (int i = threadIdx.x; i < WN * MR * 16; i += W4_WAVES * 64) {
            const int j = i & 15, mm = (i >> 4) % MR, t = (i >> 4) / MR, col = (set * WN + t) * 16 + j;
            float v = rp[((t << a.wk_log) * MR + mm) * 16 + j];
            for (int k = 1; k < WK; k++) v += rp[(((t << a.wk_log) + k) * MR + mm) * 16 + j];
            if (col < a.n && row0 + mm < a.rows) a.y[(long long) (row0 + mm) * a.y_stride + col] = v;
        }
    }
}

constexpr int W4_LDS = 64 * 1024;

template <int MODE, int DT, int NR, int RG>
static hipError_t launch_k(W4Args a, hipStream_t st) {
    constexpr int MR = NR * RG, per = planes(MODE) * MR * 16 + 2 * MR * 4;
    const int nb4 = (a.k / 32 + 3) & ~3, tiles = (a.n + 15) / 16;
    const int red = 2 * W4_WAVES * MR * 16 * 4, zero = planes(MODE) * MR * 16;
    a.kcb = std::min(nb4, ((W4_LDS - red - zero) / per) & ~3);
    while (a.wk_log < 3 && (tiles << a.wk_log) < 2048) a.wk_log++;
    const int wn = W4_WAVES >> a.wk_log, sets = (tiles + wn - 1) / wn;
    const size_t lds = (size_t) a.kcb * per + zero + red;
    hipLaunchKernelGGL((k_w4<MODE, DT, NR, RG>), dim3(std::min(sets, 512), (a.rows + MR - 1) / MR), dim3(W4_WAVES * 64), lds, st, a);
    return hipGetLastError();
}

template <int MODE, int DT>
static hipError_t launch_mode(const W4Args & a, hipStream_t st) {
    if (a.rows == 1) return launch_k<MODE, DT, 1, 1>(a, st);
    if (a.rows == 2) return launch_k<MODE, DT, 2, 1>(a, st);
    if (a.rows <= 4) return launch_k<MODE, DT, 4, 1>(a, st);
    if (a.rows <= 8) return launch_k<MODE, DT, 4, 2>(a, st);
    return launch_k<MODE, DT, 4, 4>(a, st);
}

hipError_t launch_w4(const W4Args & a, int xform, hipStream_t st) {
    switch (xform) {
    case W4_UNITS: return launch_mode<XM_UNITS, DT_F32>(a, st);
    case DT_F16: return launch_mode<XM_HALF, DT_F16>(a, st);
    case DT_BF16: return launch_mode<XM_HALF, DT_BF16>(a, st);
    default: return launch_mode<XM_SPLIT, DT_F32>(a, st);
    }
}

} // namespace qkv
