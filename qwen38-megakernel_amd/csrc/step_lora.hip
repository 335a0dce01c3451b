// Low-rank adapters of many requests at once: y[m] = base[m] + s_a B_a (A_a x[m]) with a = ids[m], next to a projection whose
// result base is.  Two kernels: u = A x of each row (a tile of 16 rows, the adapters in it one after another or side by
// side in workgroups of their own), then y = base + B u.  A row belongs to one adapter, so a tile's rows are split among
// its adapters; nothing is sorted, and an adapter's weights are read once per tile that has it.
//
// Matrix instructions take 16-bit operands and add in fp32.  Where x or u has more bits it goes in as several bf16 parts
// (truncated, 8 bits each: fp32 is three of them exactly, fp16 two), fp16 adapters as two; x of int8 units goes in as its codes,
// whose block scale (the blocks have the length of a step) multiplies the step's result.
#include "step_dev.h"
#include "step_mix_launch.h"

#include <algorithm>

namespace qkv {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// operands of a step: 8 values of a lane as `parts` 16-bit vectors
constexpr bool f16_mfma(int xf, int wf) { return wf == DT_F16 && (xf == DT_F16 || xf == W4_UNITS); }
constexpr int x_parts(int xf, int wf) { return xf == DT_F32 ? 3 : xf == DT_F16 && wf != DT_F16 ? 2 : 1; }
constexpr int w_parts(int xf, int wf) { return wf == DT_F16 && !f16_mfma(xf, wf) ? 2 : 1; }

// v as P bf16 parts, each what is left of the ones before cut to 8 bits; an infinity or a NaN is the first part's alone
template <int P> __device__ __forceinline__ void split(const float (&v)[8], u32x4 (&p)[P]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = v[i];
#pragma unroll
    for (int q = 0; q < P; q++) {
        unsigned h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            h[i] = __builtin_bit_cast(unsigned, r[i]) & 0xffff0000u;
            if (q == 0 && r[i] != r[i]) h[i] = 0x7fc00000u;
            if (q + 1 < P) r[i] = (h[i] & 0x7f800000u) == 0x7f800000u ? 0.f : r[i] - __builtin_bit_cast(float, h[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) p[q][i] = h[2 * i] >> 16 | h[2 * i + 1];
    }
}

template <bool F16> __device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// an adapter's 8 weights as they are in memory -> the operand's parts
template <int WF, int P> __device__ __forceinline__ void open_w(u32x4 raw, u32x4 (&p)[P]) {
    if constexpr (P == 1) p[0] = raw;
    else {
        float v[8];
        Elem<DT_F16>::open8(__builtin_bit_cast(half8, raw), v);
        split<P>(v, p);
    }
}

// the adapters of a tile of 16 rows, one after another: a's rows in lanes (row n = lane & 15) of `mine`
struct Adapters {
    unsigned todo; // rows whose adapter is still to come
    int id;        // the lane's row's
    bool has;
    __device__ __forceinline__ Adapters(const LoraArgs & a, int row) {
        id = row < a.rows ? a.ids[row] : -1;
        has = (unsigned) id < (unsigned) a.n_adapters;
        todo = (unsigned) __ballot(has) & 0xffffu;
    }
    // the next one, or -1
    __device__ __forceinline__ int next(bool & mine) {
        if (!todo) return -1;
        const int at = __builtin_amdgcn_readlane(id, __builtin_ctz(todo));
        mine = has && id == at;
        todo &= ~(unsigned) __ballot(mine);
        return at;
    }
};
__device__ __forceinline__ int rank_of(const LoraArgs & a, int id) { return a.ranks ? min(max(a.ranks[id], 0), a.rank) : a.rank; }

constexpr int LW = 8; // waves of a workgroup of k_lora_down

// u[chunk][m][i] = sum over the chunk's k of A[ids[m]][i][k] x[m][k].  A workgroup per (tile, adapter's place, chunk); its waves take every
// LW-th step of 32 values each and add up in LDS; NT tiles of 16 ranks at a time.
template <int XF, int WF, int NT> __global__ __launch_bounds__(LW * 64) void k_lora_down(LoraArgs a) {
    constexpr bool F16 = f16_mfma(XF, WF), UNITS = XF == W4_UNITS;
    constexpr int PX = x_parts(XF, WF), PW = w_parts(XF, WF), U = NT == 1 ? 4 : 2;
    constexpr int XT = UNITS ? DT_F16 : XF; // (units: not used)
    __shared__ __attribute__((aligned(16))) float red[LW * NT * 256];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.x * 16, row = row0 + n, nb = a.k >> 5;
    const int s0 = (int) ((long long) nb * blockIdx.z / a.chunks), s1 = (int) ((long long) nb * (blockIdx.z + 1) / a.chunks);
    Adapters ad(a, row);
    bool mine;
    int place = 0;
    for (int id = ad.next(mine); id >= 0; id = ad.next(mine), place++) {
        if (place % a.slots != (int) blockIdx.y) continue;
        const int rk = rank_of(a, id);
        for (int t0 = 0; t0 < rk; t0 += 16 * NT) {
            const uint16_t * wp = static_cast<const uint16_t *>(a.a) + (size_t) id * a.rank * a.k;
            f32x4 acc[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int s = s0 + wave; s < s1; s += LW * U) {
                u32x4 w[U][NT];
                typename Elem<XT>::Raw8 xr[U];
                u32x2 xq[U];
                float xd[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int st = s + LW * u;
                    if (st >= s1) break;
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        if (t0 + 16 * t < rk) // (ranks past the last one: its row again, not stored)
                            w[u][t] = __builtin_bit_cast(u32x4, *reinterpret_cast<const u16x8_u *>(wp + (size_t) min(t0 + 16 * t + n, rk - 1) * a.k + 32 * st + 8 * g));
                    xr[u] = typename Elem<XT>::Raw8{};
                    xq[u] = u32x2{0, 0};
                    xd[u] = 0.f;
                    if (mine) {
                        if constexpr (UNITS) {
                            const size_t unit = (size_t) row * nb + (st & ~1);
                            xq[u] = *reinterpret_cast<const u32x2 *>((st & 1 ? a.xb : a.xa) + (unit + (g >> 1)) * 16 + 8 * (g & 1));
                            xd[u] = h2f_bits(a.xmeta[unit * 4 + (st & 1)]);
                        } else xr[u] = Elem<XT>::raw8(static_cast<const typename Elem<XT>::T *>(a.x) + row * a.x_stride + 32 * st + 8 * g);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (s + LW * u >= s1) break;
                    u32x4 xp[PX];
                    if constexpr (UNITS) {
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) v[i] = (float) (int8_t) (xq[u][i >> 2] >> 8 * (i & 3));
                        if constexpr (F16) {
                            half8 h;
#pragma unroll
                            for (int i = 0; i < 8; i++) h[i] = (_Float16) v[i];
                            xp[0] = __builtin_bit_cast(u32x4, h);
                        } else split<1>(v, xp); // (7 bits and a sign: exact)
                    } else if constexpr (PX == 1) xp[0] = __builtin_bit_cast(u32x4, xr[u]);
                    else {
                        float v[8];
                        Elem<XT>::open8(xr[u], v);
                        split<PX>(v, xp);
                    }
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        if (t0 + 16 * t >= rk) break;
                        u32x4 p[PW];
                        open_w<WF>(w[u][t], p);
                        f32x4 c = UNITS ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[t];
                        // small parts first; the third of x times the second of A is below 2^-24 of the product
#pragma unroll
                        for (int q = PW - 1; q >= 0; q--)
#pragma unroll
                            for (int i = PX - 1; i >= 0; i--)
                                if (i + q <= 2) c = mfma32<F16>(p[q], xp[i], c);
                        if constexpr (UNITS) {
#pragma unroll
                            for (int r = 0; r < 4; r++) acc[t][r] = __builtin_fmaf(xd[u], c[r], acc[t][r]);
                        } else acc[t] = c;
                    }
                }
            }
            __syncthreads(); // (the sums before are read)
#pragma unroll
            for (int t = 0; t < NT; t++) *reinterpret_cast<f32x4 *>(red + ((wave * NT + t) * 16 + n) * 16 + 4 * g) = acc[t];
            __syncthreads();
            // rows of the adapter, one of its ranks a thread
            const unsigned of = (unsigned) __ballot(mine) & 0xffffu;
            for (int i = threadIdx.x; i < NT * 256; i += LW * 64) {
                const int m = i >> 4 & 15, r = t0 + (i >> 8) * 16 + (i & 15);
                if (!(of >> m & 1) || r >= rk) continue;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < LW; w++) v += red[w * NT * 256 + i];
                a.u[((size_t) blockIdx.z * a.rows + row0 + m) * a.rp + r] = v;
            }
        }
    }
}

constexpr int UW = 4; // waves of a workgroup of k_lora_up

// y = base + s B u: a wave takes CT tiles of 16 columns of a tile of 16 rows; the adapters of the tile split its rows.  u in three bf16
// parts, whose products with B add up in fp32 (fp16 B: two parts).
template <int WF, int CT> __global__ __launch_bounds__(UW * 64) void k_lora_up(LoraArgs a) {
    constexpr int PW = WF == DT_F16 ? 2 : 1;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int row = blockIdx.y * 16 + n, c0 = (blockIdx.x * UW + wave) * CT * 16;
    if (c0 >= a.n) return;
    Adapters ad(a, row);
    // y of the lane's row, columns c0 + 16 t + 4 g on
    const auto store = [&](const f32x4 (&acc)[CT]) {
#pragma unroll
        for (int t = 0; t < CT; t++) {
            const int c = c0 + 16 * t + 4 * g;
            float * y = a.y + row * a.y_stride + c;
            const float * b = a.base ? a.base + row * a.base_stride + c : nullptr;
            if (c + 4 <= a.n) {
                f32x4 v = acc[t];
                if (b) v += *reinterpret_cast<const f32x4_u *>(b);
                *reinterpret_cast<f32x4_u *>(y) = v;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (c + i < a.n) y[i] = b ? b[i] + acc[t][i] : acc[t][i];
            }
        }
    };
    f32x4 acc[CT];
    if (blockIdx.z == 0 && row < a.rows && !ad.has) {
#pragma unroll
        for (int t = 0; t < CT; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        store(acc);
    }
    bool mine;
    int place = 0;
    for (int id = ad.next(mine); id >= 0; id = ad.next(mine), place++) {
        if (place % a.slots != (int) blockIdx.z) continue;
        const int rk = rank_of(a, id);
        const float sc = a.scales ? a.scales[id] : 1.f;
        const uint16_t * bp = static_cast<const uint16_t *>(a.b) + (size_t) id * a.n * a.rank;
#pragma unroll
        for (int t = 0; t < CT; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int r0 = 0; r0 < rk; r0 += 32) {
            const int r = r0 + 8 * g;
            u32x4 raw[CT];
#pragma unroll
            for (int t = 0; t < CT; t++) {
                const uint16_t * p = bp + (size_t) min(c0 + 16 * t + n, a.n - 1) * a.rank + r;
                raw[t] = u32x4{0, 0, 0, 0};
                if (r + 8 <= rk) raw[t] = __builtin_bit_cast(u32x4, *reinterpret_cast<const u16x8_u *>(p));
                else if (r < rk) {
                    unsigned e[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) e[i] = r + i < rk ? p[i] : 0;
                    raw[t] = u32x4{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
                }
            }
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0.f;
            if (mine && r < rk) {
                for (int c = 0; c < a.chunks; c++) { // (rows of u are padded to 16 ranks)
                    const float * up = a.u + ((size_t) c * a.rows + row) * a.rp + r;
                    const f32x4 lo = *reinterpret_cast<const f32x4 *>(up), hi = *reinterpret_cast<const f32x4 *>(up + 4);
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] += lo[i], v[4 + i] += hi[i];
                }
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = r + i < rk ? v[i] * sc : 0.f;
            }
            u32x4 up[3];
            split<3>(v, up);
#pragma unroll
            for (int t = 0; t < CT; t++) {
                u32x4 p[PW];
                open_w<WF>(raw[t], p);
#pragma unroll
                for (int q = PW - 1; q >= 0; q--)
#pragma unroll
                    for (int i = 2; i >= 0; i--)
                        if (i + q <= 2) acc[t] = mfma32<false>(p[q], up[i], acc[t]);
            }
        }
        if (mine) store(acc);
    }
}

template <int XF, int WF> hipError_t down(const LoraArgs & a, hipStream_t st) {
    const dim3 grid((a.rows + 15) / 16, a.slots, a.chunks), block(LW * 64);
    return a.rank <= 16 ? launch(k_lora_down<XF, WF, 1>, grid, block, 0, st, a) : launch(k_lora_down<XF, WF, 4>, grid, block, 0, st, a);
}
template <int WF, int CT> hipError_t up(const LoraArgs & a, hipStream_t st) {
    return launch(k_lora_up<WF, CT>, dim3((a.n + 16 * CT * UW - 1) / (16 * CT * UW), (a.rows + 15) / 16, a.slots), dim3(UW * 64), 0, st, a);
}

} // namespace

void lora_plan(LoraArgs & a) {
    const int tiles = (a.rows + 15) / 16, steps = a.k / 32;
    a.rp = (a.rank + 15) / 16 * 16;
    // few tiles: the adapters of a tile in workgroups of their own
    a.slots = a.rows <= 256 ? std::min(16, std::max(a.rows, 1)) : 1;
    // and k in chunks, of at least four steps a wave, until two workgroups a CU have work
    const int busy = std::max(1, tiles * a.slots);
    a.chunks = std::max(1, std::min({LORA_MAX_CHUNKS, 512 / busy, steps / (4 * LW)}));
}

hipError_t launch_lora(const LoraArgs & a, int xform, int wtype, hipStream_t st) {
    hipError_t e;
    if (wtype == DT_F16)
        e = xform == W4_UNITS ? down<W4_UNITS, DT_F16>(a, st) : xform == DT_F32 ? down<DT_F32, DT_F16>(a, st) : xform == DT_F16 ? down<DT_F16, DT_F16>(a, st) : down<DT_BF16, DT_F16>(a, st);
    else
        e = xform == W4_UNITS ? down<W4_UNITS, DT_BF16>(a, st) : xform == DT_F32 ? down<DT_F32, DT_BF16>(a, st) : xform == DT_F16 ? down<DT_F16, DT_BF16>(a, st) : down<DT_BF16, DT_BF16>(a, st);
    if (e != hipSuccess) return e;
    // 64 columns a wave where that leaves a wave for every SIMD
    const bool wide = (long long) ((a.n + 63) / 64) * ((a.rows + 15) / 16) >= 1024;
    if (wtype == DT_F16) return wide ? up<DT_F16, 4>(a, st) : up<DT_F16, 1>(a, st);
    return wide ? up<DT_BF16, 4>(a, st) : up<DT_BF16, 1>(a, st);
}

} // namespace qkv
