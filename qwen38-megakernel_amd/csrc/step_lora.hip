// Low-rank adapters of many requests at once: y[m] = base[m] + s_a B_a (A_a x[m]) with a = ids[m], next to a projection whose
// result base is.  Two kernels: u = A x of each row, then y = base + B u.  Nothing is sorted: a workgroup has a tile of 16 rows (32 of
// many) and takes the adapters in it one after another, or, where tiles are few, side by side in workgroups of their own; a row belongs
// to one adapter, so a tile's rows are split among its adapters.
//
// Matrix instructions take 16-bit operands and add in fp32.  The adapters' weights go in as they are.  Where x has more bits than their type it
// goes in as several parts: bf16 adapters take fp16 x as two bf16 parts and fp32 x as three (truncated, 8 bits each: exact); fp16
// adapters take bf16 x as one and fp32 x as two fp16 parts after a power of two per row and step of 32 values, which multiplies the step's
// result (2^-39 and 2^-23 of the largest of the 32).  Int8 units go in as their codes, the block's scale multiplying the step's result.  u goes in
// as three bf16 parts, or two fp16 parts after a power of two per row and 64 ranks.
//
// Memory bounds it at every size (4 rank operations for 2 bytes of an adapter, and 8 bytes of base and y a column).  1 fp32 row of 5,120 x 6,144 and
// rank 16: 9.3 us, two launches and their chains of loads (in one launch, every workgroup computing u for itself, a bf16 row takes 10.4 where two take
// 7.8).  61 rows of as many fp16 adapters of ranks up to 64, 17,408 x 5,120: 54 us, of them 36 for B, 2.9 TB/s.  4,001 rows of 6,144 x 5,120
// and rank 32: 78 us, of them 56 for 197 MB of base and y.
#include "step_dev.h"
#include "step_mix_launch.h"

#include <algorithm>
#include <type_traits>

namespace qkv {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <int WF> __device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (WF == DT_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// v as P bf16 parts, each what is left of the ones before cut to 8 bits; an infinity or a NaN is the first part's alone
template <int P> __device__ __forceinline__ void split_bf16(const float (&v)[8], u32x4 (&p)[P]) {
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
// The four lane groups' values of a row times 2^e, which brings the largest (its bits: top) to [2^14, 2^15), as P fp16 parts; returns 2^-e.
// Beside an infinity or a NaN finite values are zeros (they cannot change the result).
template <int P> __device__ __forceinline__ float split_f16(float (&v)[8], unsigned top, u32x4 (&p)[P]) {
    const bool wild = top >= 0x7f800000u;
    const int E = max((int) (top >> 23), 15);
    const float up = __builtin_bit_cast(float, (unsigned) (268 - E) << 23);
    half8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float w = !wild ? v[i] * up : __builtin_fabsf(v[i]) < __builtin_inff() ? 0.f : v[i];
        hi[i] = (_Float16) w;
        lo[i] = (_Float16) (wild ? 0.f : w - (float) hi[i]);
    }
    p[0] = __builtin_bit_cast(u32x4, hi);
    if constexpr (P > 1) p[1] = __builtin_bit_cast(u32x4, lo);
    return wild ? 1.f : __builtin_bit_cast(float, (unsigned) (E - 14) << 23);
}
__device__ __forceinline__ unsigned row_top(unsigned t) { // over the four lane groups
    t = max(t, shfl_xor_u(t, 16));
    return max(t, shfl_xor_u(t, 32));
}

// the adapters of a tile of RT x 16 rows, one after another: lane n = lane & 15 has rows n, 16 + n
template <int RT> struct Adapters {
    unsigned todo; // rows whose adapter is still to come
    int id[RT];
    bool has[RT];
    __device__ __forceinline__ Adapters(const LoraArgs & a, int row) {
        todo = 0;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            id[t] = row + 16 * t < a.rows ? a.ids[row + 16 * t] : -1;
            has[t] = (unsigned) id[t] < (unsigned) a.n_adapters;
            todo |= ((unsigned) __ballot(has[t]) & 0xffffu) << 16 * t;
        }
    }
    // the next one and its rows, or -1
    __device__ __forceinline__ int next(bool (&mine)[RT]) {
        if (!todo) return -1;
        const int b = __builtin_ctz(todo);
        int at = __builtin_amdgcn_readlane(id[0], b & 15);
        if constexpr (RT == 2)
            if (b > 15) at = __builtin_amdgcn_readlane(id[1], b & 15);
#pragma unroll
        for (int t = 0; t < RT; t++) {
            mine[t] = has[t] && id[t] == at;
            todo &= ~(((unsigned) __ballot(mine[t]) & 0xffffu) << 16 * t);
        }
        return at;
    }
};
__device__ __forceinline__ int rank_of(const LoraArgs & a, int id) { return a.ranks ? min(max(a.ranks[id], 0), a.rank) : a.rank; }

constexpr int LW = 8; // waves of a workgroup of k_lora_down

constexpr bool scaled(int xf, int wf) { return xf == W4_UNITS || (wf == DT_F16 && xf != DT_F16); } // a step's result has a factor of its own
constexpr int x_parts(int xf, int wf) { return xf == DT_F32 ? (wf == DT_F16 ? 2 : 3) : xf == DT_F16 && wf != DT_F16 ? 2 : 1; }

// u[chunk][m][i] = sum over the chunk's k of A[ids[m]][i][k] x[m][k].  A workgroup per (tile, adapter's place, chunk); its waves take every
// LW-th pair of steps of 32 values each (a cache line of every row), one or two pairs' loads at a time, and add up in LDS; NT tiles of 16 ranks
// at a time.
template <int XF, int WF, int NT, int RT> __global__ __launch_bounds__(LW * 64) void k_lora_down(LoraArgs a) {
    constexpr bool UNITS = XF == W4_UNITS, SCALED = scaled(XF, WF);
    constexpr int PX = x_parts(XF, WF), U = NT == 4 ? 2 : 4; // (registers for two workgroups a CU)
    constexpr int XT = UNITS ? DT_F16 : XF; // (units: not used)
    __shared__ __attribute__((aligned(16))) float red[LW * RT * NT * 256];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.x * 16 * RT, row = row0 + n, nb = a.k >> 5, np = (nb + 1) >> 1;
    const int p0 = (int) ((long long) np * blockIdx.z / a.chunks), p1 = (int) ((long long) np * (blockIdx.z + 1) / a.chunks);
    Adapters<RT> ad(a, row);
    bool mine[RT];
    int place = 0;
    for (int id = ad.next(mine); id >= 0; id = ad.next(mine), place++) {
        if (a.slots > 1 && place != (int) blockIdx.y) continue; // (as many places as a tile has rows, or one workgroup for all)
        const int rk = rank_of(a, id);
        for (int t0 = 0; t0 < rk; t0 += 16 * NT) {
            const uint16_t * wp = static_cast<const uint16_t *>(a.a) + (size_t) id * a.rank * a.k;
            f32x4 acc[RT][NT];
#pragma unroll
            for (int q = 0; q < RT; q++)
#pragma unroll
                for (int t = 0; t < NT; t++) acc[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int p = p0 + wave; p < p1; p += LW * (U / 2)) {
                u32x4 w[U][NT];
                typename Elem<XT>::Raw8 xr[U][RT];
                u32x2 xq[U][RT];
                float xd[U][RT];
                const auto step = [&](int u) { return 2 * (p + LW * (u >> 1)) + (u & 1); };
                const auto in = [&](int u) { return p + LW * (u >> 1) < p1 && step(u) < nb; };
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (!in(u)) continue;
                    const int st = step(u);
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        if (t0 + 16 * t < rk) // (ranks past the last one: its row again, not stored)
                            w[u][t] = __builtin_bit_cast(u32x4, *reinterpret_cast<const u16x8_u *>(wp + (size_t) min(t0 + 16 * t + n, rk - 1) * a.k + 32 * st + 8 * g));
#pragma unroll
                    for (int q = 0; q < RT; q++) {
                        xr[u][q] = typename Elem<XT>::Raw8{};
                        xq[u][q] = u32x2{0, 0};
                        xd[u][q] = 0.f;
                        if (!mine[q]) continue;
                        const int r = row + 16 * q;
                        if constexpr (UNITS) {
                            const size_t unit = (size_t) r * nb + (st & ~1);
                            xq[u][q] = *reinterpret_cast<const u32x2 *>((st & 1 ? a.xb : a.xa) + (unit + (g >> 1)) * 16 + 8 * (g & 1));
                            xd[u][q] = h2f_bits(a.xmeta[unit * 4 + (st & 1)]);
                        } else xr[u][q] = Elem<XT>::raw8(static_cast<const typename Elem<XT>::T *>(a.x) + r * a.x_stride + 32 * st + 8 * g);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (!in(u)) continue;
#pragma unroll
                    for (int q = 0; q < RT; q++) {
                        u32x4 xp[PX];
                        float d = xd[u][q];
                        if constexpr (UNITS) {
                            float v[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) v[i] = (float) (int8_t) (xq[u][q][i >> 2] >> 8 * (i & 3));
                            if constexpr (WF == DT_F16) {
                                half8 h;
#pragma unroll
                                for (int i = 0; i < 8; i++) h[i] = (_Float16) v[i];
                                xp[0] = __builtin_bit_cast(u32x4, h);
                            } else split_bf16<1>(v, xp); // (7 bits and a sign: exact)
                        } else if constexpr (SCALED) {
                            float v[8];
                            Elem<XT>::open8(xr[u][q], v);
                            d = split_f16<PX>(v, row_top(Elem<XT>::top8(xr[u][q])), xp);
                        } else if constexpr (PX == 1) xp[0] = __builtin_bit_cast(u32x4, xr[u][q]);
                        else {
                            float v[8];
                            Elem<XT>::open8(xr[u][q], v);
                            split_bf16<PX>(v, xp);
                        }
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            if (t0 + 16 * t >= rk) continue;
                            f32x4 c = SCALED ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[q][t];
#pragma unroll
                            for (int i = PX - 1; i >= 0; i--) c = mfma32<WF>(w[u][t], xp[i], c); // (small parts first)
                            if constexpr (SCALED) {
#pragma unroll
                                for (int r = 0; r < 4; r++) acc[q][t][r] = __builtin_fmaf(d, c[r], acc[q][t][r]);
                            } else acc[q][t] = c;
                        }
                    }
                }
            }
            __syncthreads(); // (the sums before are read)
#pragma unroll
            for (int q = 0; q < RT; q++)
#pragma unroll
                for (int t = 0; t < NT; t++) *reinterpret_cast<f32x4 *>(red + (((wave * RT + q) * NT + t) * 16 + n) * 16 + 4 * g) = acc[q][t];
            __syncthreads();
            // rows of the adapter, one of its ranks a thread
            unsigned of[RT];
#pragma unroll
            for (int q = 0; q < RT; q++) of[q] = (unsigned) __ballot(mine[q]) & 0xffffu;
            for (int i = threadIdx.x; i < RT * NT * 256; i += LW * 64) {
                const int q = RT == 1 ? 0 : i / (NT * 256), m = i >> 4 & 15, r = t0 + (i >> 8) % NT * 16 + (i & 15);
                if (!((q ? of[RT - 1] : of[0]) >> m & 1) || r >= rk) continue;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < LW; w++) v += red[w * RT * NT * 256 + i];
                a.u[((size_t) blockIdx.z * a.rows + row0 + 16 * q + m) * a.rp + r] = v;
            }
        }
    }
}

constexpr int UW = 4, UP_WAVES = 12 * 256; // waves of a workgroup of k_lora_up; of its grid, where the groups of columns are more

// y = base + s B u: a wave has u of a tile's rows in registers (KH x 32 ranks of it; ranks past 64: 64 at a time, of every group anew) and takes
// its share of the groups of CT x 16 columns, the next group's B and base on their way.
template <int WF, int CT, int RT, int KH, bool BIG> __global__ __launch_bounds__(UW * 64, 3) void k_lora_up(LoraArgs a) {
    constexpr int PU = WF == DT_F16 ? 2 : 3;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int row = blockIdx.y * 16 * RT + n, waves0 = gridDim.x * UW, wave0 = blockIdx.x * UW + wave, groups = (a.n + 16 * CT - 1) / (16 * CT);
    Adapters<RT> ad(a, row);
    // y of rows row + 16 q, four columns from c on
    const auto load = [&](int q, int c) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (!a.base) return v;
        const float * b = a.base + (row + 16 * q) * a.base_stride + c;
        if (c + 4 <= a.n) return f32x4(*reinterpret_cast<const f32x4_u *>(b));
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (c + i < a.n) v[i] = b[i];
        return v;
    };
    const auto store = [&](int q, int c, f32x4 v) {
        float * y = a.y + (row + 16 * q) * a.y_stride + c;
        if (c + 4 <= a.n) *reinterpret_cast<f32x4_u *>(y) = v;
        else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (c + i < a.n) y[i] = v[i];
        }
    };
    // the tile's adapters share its waves: wave w has the (w mod D)-th of D, and those that have it share the columns
    bool mine[RT];
    int adapters = 0;
    for (Adapters<RT> all = ad; all.next(mine) >= 0;) adapters++;
    const int own = adapters ? wave0 % adapters : 0, first = adapters <= waves0 ? (adapters ? wave0 / adapters : wave0) : 0;
    const int step = adapters <= waves0 ? (adapters ? (waves0 - own + adapters - 1) / adapters : waves0) : 1;
    // rows without an adapter: base as it is
    if (a.base != a.y) {
#pragma unroll
        for (int q = 0; q < RT; q++) {
            const bool none = row + 16 * q < a.rows && !ad.has[q];
            if (!__ballot(none)) continue;
            for (int cg = wave0; cg < groups; cg += waves0)
#pragma unroll
                for (int t = 0; t < CT; t++)
                    if (none) store(q, cg * 16 * CT + 16 * t + 4 * g, load(q, cg * 16 * CT + 16 * t + 4 * g));
        }
    }
    int place = 0;
    for (int id = ad.next(mine); id >= 0; id = ad.next(mine), place++) {
        if (adapters <= waves0 ? place != own : place % waves0 != wave0) continue;
        const int rk = rank_of(a, id);
        const float sc = a.scales ? a.scales[id] : 1.f;
        const uint16_t * bp = static_cast<const uint16_t *>(a.b) + (size_t) id * a.n * a.rank;
        // rows of others stand for the adapter's first one: loads, results and stores are the same, and no branch is in the loop, where the compiler
        // would wait for the loads of the next group with this one's
        unsigned rows = 0;
#pragma unroll
        for (int q = 0; q < RT; q++) rows |= ((unsigned) __ballot(mine[q]) & 0xffffu) << 16 * q;
        long long at[RT];
#pragma unroll
        for (int q = 0; q < RT; q++) at[q] = mine[q] ? row + 16 * q : (int) blockIdx.y * 16 * RT + __builtin_ctz(rows);
        u32x4 up[RT][KH][PU];
        float back[RT];
        const auto parts = [&](int r0) { // ranks r0 .. r0 + 32 KH - 1 of u
#pragma unroll
            for (int q = 0; q < RT; q++) {
                float v[KH][8];
                unsigned top = 0;
#pragma unroll
                for (int h = 0; h < KH; h++) {
                    const int r = r0 + 32 * h + 8 * g;
#pragma unroll
                    for (int i = 0; i < 8; i++) v[h][i] = 0.f;
                    if (r < a.rp) { // (rows of u are padded to 16 ranks; what lies past rk is left out below)
                        const float * ur = a.u + (size_t) at[q] * a.rp + r;
                        const size_t chunk = (size_t) a.rows * a.rp;
                        for (int c0 = 0; c0 < a.chunks; c0 += 4) { // (four loads, then their sums)
                            f32x4 lo[4], hi[4];
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                const float * p = ur + min(c0 + c, a.chunks - 1) * chunk;
                                lo[c] = *reinterpret_cast<const f32x4 *>(p);
                                hi[c] = *reinterpret_cast<const f32x4 *>(p + 4);
                            }
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                if (c0 + c < a.chunks) {
#pragma unroll
                                    for (int i = 0; i < 4; i++) v[h][i] += lo[c][i], v[h][4 + i] += hi[c][i];
                                }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        v[h][i] = r + i < rk ? v[h][i] * sc : 0.f;
                        top = max(top, __builtin_bit_cast(unsigned, v[h][i]) & 0x7fffffffu);
                    }
                }
                back[q] = 1.f;
                if constexpr (WF == DT_F16) {
                    top = row_top(top);
#pragma unroll
                    for (int h = 0; h < KH; h++) back[q] = split_f16<PU>(v[h], top, up[q][h]);
                } else {
#pragma unroll
                    for (int h = 0; h < KH; h++) split_bf16<PU>(v[h], up[q][h]);
                }
            }
        };
        // 8 ranks of a row of B from r on, the elements past rk zeros; where the row ends before them its last 8 elements, moved down
        const auto weights = [&](int cg, int r0, u32x4 (&raw)[CT][KH]) {
#pragma unroll
            for (int h = 0; h < KH; h++) {
                const int r = r0 + 32 * h + 8 * g, over = max(r + 8 - a.rank, 0), left = rk - r;
                u32x4 mask;
#pragma unroll
                for (int i = 0; i < 4; i++) mask[i] = left >= 2 * i + 2 ? ~0u : left == 2 * i + 1 ? 0xffffu : 0;
#pragma unroll
                for (int t = 0; t < CT; t++) {
                    const uint16_t * p = bp + (size_t) min(cg * 16 * CT + 16 * t + n, a.n - 1) * a.rank + r;
                    u32x4 v = {0, 0, 0, 0};
                    if (a.rank < 8) {
                        if (left > 0) {
                            unsigned e[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) e[i] = i < left ? p[i] : 0;
                            v = u32x4{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
                        }
                    } else if (left > 0) {
                        v = __builtin_bit_cast(u32x4, *reinterpret_cast<const u16x8_u *>(p - over));
                        if (a.rank & 7) {
                            if (over & 4) v = u32x4{v[2], v[3], 0, 0};
                            if (over & 2) v = u32x4{v[1], v[2], v[3], 0};
                            if (over & 1) v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
                        }
                    }
                    raw[t][h] = v & mask;
                }
            }
        };
        const auto bases = [&](int cg, f32x4 (&y)[RT][CT]) {
#pragma unroll
            for (int q = 0; q < RT; q++)
#pragma unroll
                for (int t = 0; t < CT; t++) y[q][t] = mine[q] ? load(q, cg * 16 * CT + 16 * t + 4 * g) : f32x4{0.f, 0.f, 0.f, 0.f};
        };
        const auto add = [&](int r0, const u32x4 (&raw)[CT][KH], f32x4 (&y)[RT][CT]) {
#pragma unroll
            for (int q = 0; q < RT; q++)
#pragma unroll
                for (int t = 0; t < CT; t++) {
                    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = KH - 1; h >= 0; h--) {
                        if (r0 + 32 * h >= rk) continue;
#pragma unroll
                        for (int i = PU - 1; i >= 0; i--) c = mfma32<WF>(raw[t][h], up[q][h][i], c); // (small parts first)
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) y[q][t][i] = __builtin_fmaf(back[q], c[i], y[q][t][i]);
                }
        };
        const auto stores = [&](int cg, const f32x4 (&y)[RT][CT]) {
#pragma unroll
            for (int q = 0; q < RT; q++)
#pragma unroll
                for (int t = 0; t < CT; t++)
                    if (mine[q]) store(q, cg * 16 * CT + 16 * t + 4 * g, y[q][t]);
        };
        if (first >= groups) continue;
        u32x4 raw[2][CT][KH];
        f32x4 y[2][RT][CT];
        if constexpr (BIG) {
            for (int cg = first; cg < groups; cg += step) {
                bases(cg, y[0]);
                f32x4 sum[RT][CT] = {};
                for (int r0 = 0; r0 < rk; r0 += 32 * KH) {
                    weights(cg, r0, raw[0]);
                    parts(r0);
                    add(r0, raw[0], sum);
                }
#pragma unroll
                for (int q = 0; q < RT; q++)
#pragma unroll
                    for (int t = 0; t < CT; t++) y[0][q][t] += sum[q][t];
                stores(cg, y[0]);
            }
        } else {
            // groups of whole columns
            const int whole = a.rank >= 8 ? a.n / (16 * CT) : 0;
            const uint16_t * wq[KH];
            u32x4 mask[KH];
            int over[KH];
#pragma unroll
            for (int h = 0; h < KH; h++) {
                const int r = 32 * h + 8 * g;
                over[h] = max(r + 8 - a.rank, 0);
                wq[h] = bp + (size_t) n * a.rank + r - over[h];
#pragma unroll
                for (int i = 0; i < 4; i++) mask[h][i] = rk - r >= 2 * i + 2 ? ~0u : rk - r == 2 * i + 1 ? 0xffffu : 0;
            }
            const auto fetch = [&](int cg, int b, auto with_base) {
#pragma unroll
                for (int h = 0; h < KH; h++)
#pragma unroll
                    for (int t = 0; t < CT; t++) raw[b][t][h] = __builtin_bit_cast(u32x4, *reinterpret_cast<const u16x8_u *>(wq[h] + (size_t) (cg * 16 * CT + 16 * t) * a.rank));
#pragma unroll
                for (int q = 0; q < RT; q++)
#pragma unroll
                    for (int t = 0; t < CT; t++) {
                        y[b][q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
                        if constexpr (decltype(with_base)::value) y[b][q][t] = f32x4(*reinterpret_cast<const f32x4_u *>(a.base + at[q] * a.base_stride + (cg * 16 * CT + 16 * t + 4 * g)));
                    }
            };
            const auto run = [&](auto with_base) {
                const auto group = [&](int cg, int b) {
                    fetch(cg + step < whole ? cg + step : cg, b ^ 1, with_base); // (behind the last group that one again, unused)
#pragma unroll
                    for (int h = 0; h < KH; h++)
#pragma unroll
                        for (int t = 0; t < CT; t++) {
                            u32x4 & v = raw[b][t][h];
                            if (a.rank & 7) {
                                if (over[h] & 4) v = u32x4{v[2], v[3], 0, 0};
                                if (over[h] & 2) v = u32x4{v[1], v[2], v[3], 0};
                                if (over[h] & 1) v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
                            }
                            v &= mask[h];
                        }
                    add(0, raw[b], y[b]);
#pragma unroll
                    for (int q = 0; q < RT; q++)
#pragma unroll
                        for (int t = 0; t < CT; t++) *reinterpret_cast<f32x4_u *>(a.y + at[q] * a.y_stride + (cg * 16 * CT + 16 * t + 4 * g)) = y[b][q][t];
                };
                for (int cg = first; cg < whole; cg += 2 * step) {
                    group(cg, 0);
                    if (cg + step < whole) group(cg + step, 1);
                }
            };
            if (first < whole) a.base ? fetch(first, 0, std::true_type()) : fetch(first, 0, std::false_type());
            parts(0);
            if (first < whole) a.base ? run(std::true_type()) : run(std::false_type());
            int cg = first < whole ? first + (whole - first + step - 1) / step * step : first;
            for (; cg < groups; cg += step) {
                weights(cg, 0, raw[0]);
                bases(cg, y[0]);
                add(0, raw[0], y[0]);
                stores(cg, y[0]);
            }
        }
    }
}

template <int XF, int WF, int RT> hipError_t down(const LoraArgs & a, hipStream_t st) {
    const dim3 grid((a.rows + 16 * RT - 1) / (16 * RT), a.slots, a.chunks), block(LW * 64);
    return a.rank <= 16 ? launch(k_lora_down<XF, WF, 1, RT>, grid, block, 0, st, a) : a.rank <= 32 ? launch(k_lora_down<XF, WF, 2, RT>, grid, block, 0, st, a)
                                                                                               : launch(k_lora_down<XF, WF, 4, RT>, grid, block, 0, st, a);
}
template <int WF, int CT, int RT> hipError_t up(const LoraArgs & a, hipStream_t st) {
    const int tiles = (a.rows + 16 * RT - 1) / (16 * RT), groups = (a.n + 16 * CT - 1) / (16 * CT);
    const int waves = std::max(1, (int) std::min<long long>((long long) groups * std::min(a.rows, 16 * RT), UP_WAVES / tiles));
    const dim3 grid((waves + UW - 1) / UW, tiles), block(UW * 64);
    if constexpr (CT == 1 || RT == 1)
        if (a.rank > 32 && a.rank <= 64) return launch(k_lora_up<WF, CT, RT, 2, false>, grid, block, 0, st, a);
    if constexpr (CT == 2 || RT == 1) return a.rank <= 32 ? launch(k_lora_up<WF, CT, RT, 1, false>, grid, block, 0, st, a) : launch(k_lora_up<WF, CT, RT, 2, true>, grid, block, 0, st, a);
    return hipErrorInvalidValue; // (not reached)
}
template <int WF, int RT> hipError_t run(const LoraArgs & a, int xform, hipStream_t st) {
    const hipError_t e = xform == W4_UNITS ? down<W4_UNITS, WF, RT>(a, st) : xform == DT_F32 ? down<DT_F32, WF, RT>(a, st) : xform == DT_F16 ? down<DT_F16, WF, RT>(a, st) : down<DT_BF16, WF, RT>(a, st);
    if (e != hipSuccess) return e;
    // (of 33 to 64 ranks two parts of u lie in the registers)
    if constexpr (RT == 2) return a.rank <= 32 || a.rank > 64 ? up<WF, 2, 2>(a, st) : up<WF, 1, 2>(a, st);
    else {
        // 32 columns a wave, a cache line of a row, where that leaves a wave for every SIMD
        const bool wide = (long long) ((a.n + 31) / 32) * ((a.rows + 15) / 16) >= 1024;
        return wide ? up<WF, 2, 1>(a, st) : up<WF, 1, 1>(a, st);
    }
}

} // namespace

void lora_plan(LoraArgs & a) {
    a.rp = (a.rank + 15) / 16 * 16;
    // few rows: the adapters of a tile in workgroups of their own; many: tiles of 32 rows, which read A and B half as often
    a.slots = a.rows <= LORA_FEW_ROWS ? std::min(16, std::max(a.rows, 1)) : 1;
    const int rt = a.rows <= LORA_FEW_ROWS ? 1 : 2, tiles = (a.rows + 16 * rt - 1) / (16 * rt), pairs = (a.k / 32 + 1) / 2;
    // and k in chunks, of at least two pairs of steps a wave, until two workgroups a CU have work
    const int busy = a.rows <= LORA_SINGLE_ROWS ? a.slots : std::min(a.slots, LORA_TILE_ADAPTERS);
    a.chunks = std::max(1, std::min({LORA_MAX_CHUNKS, 512 / std::max(1, tiles * busy), pairs / (2 * LW)}));
}

hipError_t launch_lora(const LoraArgs & a, int xform, int wtype, hipStream_t st) {
    if (wtype == DT_F16) return a.rows <= LORA_FEW_ROWS ? run<DT_F16, 1>(a, xform, st) : run<DT_F16, 2>(a, xform, st);
    return a.rows <= LORA_FEW_ROWS ? run<DT_BF16, 1>(a, xform, st) : run<DT_BF16, 2>(a, xform, st);
}

} // namespace qkv
