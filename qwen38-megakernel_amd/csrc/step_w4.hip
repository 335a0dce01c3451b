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
#include <atomic>
#include <type_traits>

namespace qkv {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4_u8 __attribute__((ext_vector_type(4), aligned(8)));

enum { XM_UNITS = 0, XM_HALF = 1, XM_SPLIT = 2 }; // x as int8 units, as one fp16 part, as two

// 16-byte planes per block of 32 values in LDS
constexpr int planes(int mode) { return mode == XM_UNITS ? 2 : mode == XM_HALF ? 4 : 8; }

// x in LDS, kcb blocks at a time.  Units, as they come: per row the even blocks' kcb units, then the odd ones', padded so that the
// 16 pieces an instruction takes (4 blocks of 4 rows) lie in different banks.  Plain rows, as fp16:
// [kcb blocks][planes][MR rows][16 bytes], fp32's two parts with 16 bytes behind every 8 blocks where k is in parts: their pieces then
// lie in different banks (2 rows of fp32 x 17,408 x 5,120: 8% less time; one row of bf16 x 150,001, half the planes: 4% more).  Then zeros for the operand's other lanes, [kcb][MR] float factors of the blocks'
// sums and (with m) [kcb][MR] float factors of m.
struct W4Lds {
    int half, row, zero, dx, ds, end; // units: bytes of a row's even blocks, of a row; offsets of the zeros, the factors, what follows
};
constexpr int run_pad(int mode, int mr) { return mode == XM_SPLIT && mr <= 2 ? 16 : 0; }
template <int MODE, int MR, bool MINS> __host__ __device__ __forceinline__ constexpr W4Lds w4_lds(int kcb) {
    W4Lds l{};
    l.half = ((kcb * 16 + 255) & ~255) + 16;
    l.row = 2 * l.half + 32;
    l.zero = MODE == XM_UNITS ? MR * l.row : kcb * planes(MODE) * MR * 16 + kcb / 8 * run_pad(MODE, MR);
    l.dx = l.zero + (MODE == XM_UNITS ? 32 : planes(MODE) * MR * 16);
    l.ds = l.dx + kcb * MR * 4;
    l.end = ((MINS ? l.ds + kcb * MR * 4 : l.ds) + 15) & ~15;
    return l;
}

// a quarter of a block of plain x (8 values) on its way to LDS as fp16: piece i = 4 (MR block + row) + quarter of the blocks from
// b0 and the rows from row0 on; zeros for rows past the last one and blocks past the row's end
template <int DT> struct W4Eighth {
    typename Elem<DT>::Raw8 raw;
    __device__ __forceinline__ void load(const W4Args & a, int i, int mr, int row0, int b0) {
        const int blk = min(b0 + (i >> 2) / mr, (a.k >> 5) - 1), row = min(row0 + (i >> 2) % mr, a.rows - 1);
        raw = Elem<DT>::raw8(static_cast<const typename Elem<DT>::T *>(a.x) + (long long) row * a.x_stride + 32 * blk + 8 * (i & 3));
    }
    // (whole blocks: the lanes of all four quarters)
    template <int MODE, int MR, bool MINS>
    __device__ __forceinline__ void store(const W4Args & a, uint8_t * lds, const W4Lds & L, int i, int row0, int b0) const {
        const int q = i & 3, m = (i >> 2) % MR, bl = (i >> 2) / MR;
        float * dx = reinterpret_cast<float *>(lds + L.dx), * ds = dx + (L.ds - L.dx) / 4;
        const bool in = row0 + m < a.rows && b0 + bl < a.k >> 5;
        float v[8], s = 0.f;
        const typename Elem<DT>::Raw8 r = in ? raw : typename Elem<DT>::Raw8{};
        unsigned top = Elem<DT>::top8(r);
        top = max(top, shfl_xor_u(top, 1));
        top = max(top, shfl_xor_u(top, 2));
        Elem<DT>::open8(r, v);
        if (MINS) {
#pragma unroll
            for (int k = 0; k < 8; k++) s += v[k];
            s += shfl_xor(s, 1);
            s += shfl_xor(s, 2);
        }
        // times 2^e, which brings the block's largest value to [2^14, 2^15), without rounding
        const bool wild = top >= 0x7f800000u;
        const int E = max((int) (top >> 23), 15);
        const float up = __builtin_bit_cast(float, (unsigned) (268 - E) << 23);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] *= up;
        if (__builtin_expect(wild, 0)) { // an infinity or a NaN in the block: these as they are, its finite values as zeros (they cannot change the result)
            Elem<DT>::open8(r, v);
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = __builtin_fabsf(v[k]) < __builtin_inff() ? 0.f : v[k];
        }
        // element order of the codes' fp16 pairs: (0, 2) (1, 3) (4, 6) (5, 7)
        half8 hi, lo;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int e = (k & 4) + 2 * (k & 1) + ((k >> 1) & 1);
            hi[e] = (_Float16) v[k];
            lo[e] = (_Float16) (v[k] - (float) hi[e]);
        }
        if (MODE == XM_SPLIT && __builtin_expect(wild, 0)) lo = half8{};
        uint8_t * to = lds + bl * (planes(MODE) * MR * 16) + (bl >> 3) * run_pad(MODE, MR) + (q * MR + m) * 16;
        *reinterpret_cast<half8 *>(to) = hi;
        if constexpr (MODE == XM_SPLIT) *reinterpret_cast<half8 *>(to + 4 * MR * 16) = lo;
        if (q == 0) {
            dx[bl * MR + m] = wild ? 1.f : __builtin_bit_cast(float, (unsigned) (E - 14) << 23);
            if (MINS) ds[bl * MR + m] = s;
        }
    }
};

// x of blocks b0 .. b0 + nblk - 1 (nblk a multiple of 4) into LDS; blocks past the last one get factors of zero
template <int MODE, int DT, int MR, int W, bool MINS>
__device__ __forceinline__ void w4_stage(const W4Args & a, uint8_t * lds, int b0, int nblk) {
    const W4Lds L = w4_lds<MODE, MR, MINS>(a.kcb);
    const int tid = threadIdx.x;
    for (int i = tid; i < (L.dx - L.zero) / 16; i += W * 64) reinterpret_cast<uint4 *>(lds + L.zero)[i] = make_uint4(0, 0, 0, 0);
    if constexpr (MODE == XM_UNITS) {
        const unsigned base = (unsigned) __builtin_amdgcn_readfirstlane((unsigned) (size_t) (__attribute__((address_space(3))) uint8_t *) lds);
        const int nb = a.k >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, np = nblk >> 1;
        float * dx = reinterpret_cast<float *>(lds + L.dx), * ds = dx + a.kcb * MR;
        // a pair of blocks' scales and sums per lane, two units of {scale a, scale b, sum a, sum b}: a wave has one row's; all
        // loads ahead of the copies, and one wait for both
        static_assert(W % MR == 0, "waves per row");
        constexpr int STEP = 64 * (W / MR), NI = 2;
        const int m = wave % MR, mrow = min(m, a.rows - 1), p0 = lane + 64 * (wave / MR);
        u32x4 mt[NI];
        const auto load = [&](int p) {
            return *reinterpret_cast<const u32x4_u8 *>(a.xmeta + ((size_t) mrow * nb + min(b0 + 2 * p, nb - 2)) * 4); // (nb is even)
        };
        const auto store = [&](int p, u32x4 v) {
            const bool in = b0 + 2 * p < nb;
            const float da = in ? h2f_bits((uint16_t) v[0]) : 0.f, db = in ? h2f_bits((uint16_t) (v[0] >> 16)) : 0.f;
            dx[2 * p * MR + m] = da * 0.0625f; // (the codes go in 16 times as large)
            dx[(2 * p + 1) * MR + m] = db * 0.0625f;
            if (MINS) {
                ds[2 * p * MR + m] = da * (float) ((int) (int16_t) v[1] + (int) (int16_t) v[3]);
                ds[(2 * p + 1) * MR + m] = db * (float) (((int) v[1] >> 16) + ((int) v[3] >> 16));
            }
        };
#pragma unroll
        for (int u = 0; u < NI; u++) mt[u] = load(min(p0 + u * STEP, np - 1));
        // 64 units of a row's even or odd blocks a copy; rows past the last one repeat it (their sums are dropped)
        const int per = (nblk + 63) >> 6; // copies of a half
#pragma unroll 1
        for (int c = wave; c < MR * 2 * per; c += W) {
            const int h = c / per, u0 = (c - h * per) * 64, row = min(h >> 1, a.rows - 1);
            if (u0 + lane < nblk)
                dma16(((h & 1) ? a.xb : a.xa) + ((size_t) row * nb + min(b0 + u0 + lane, nb - 1)) * 16,
                      base + (h >> 1) * L.row + (h & 1) * L.half + u0 * 16);
        }
#pragma unroll
        for (int u = 0; u < NI; u++)
            if (p0 + u * STEP < np) store(p0 + u * STEP, mt[u]);
        for (int p = p0 + NI * STEP; p < np; p += STEP) store(p, load(p));
        vm_drain();
    } else {
        for (int i = tid; i < nblk * 4 * MR; i += 4 * W * 64) { // (four loads, then their values)
            W4Eighth<DT> e[4];
#pragma unroll
            for (int u = 0; u < 4; u++) e[u].load(a, min(i + u * W * 64, nblk * 4 * MR - 1), MR, 0, b0);
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (i + u * W * 64 < nblk * 4 * MR) e[u].template store<MODE, MR, MINS>(a, lds, L, i + u * W * 64, 0, b0);
        }
    }
}

// the codes of one word as fp16 pairs (0, 2) (1, 3) (4, 6) (5, 7): 0x6400 | n is 1024 + n and 0x5400 | 16 n is 64 + n, both exact
__device__ __forceinline__ half8 w4_halves(unsigned w) {
    const half2v b0 = {(_Float16) -1032.f, (_Float16) -1032.f}, b1 = {(_Float16) -72.f, (_Float16) -72.f};
    const unsigned v = w >> 8;
    const half2v p0 = as_h2((w & 0x000f000fu) | 0x64006400u) + b0, p1 = as_h2((v & 0x000f000fu) | 0x64006400u) + b0,
                 p2 = as_h2((w & 0x00f000f0u) | 0x54005400u) + b1, p3 = as_h2((v & 0x00f000f0u) | 0x54005400u) + b1;
    return half8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// Plain rows with minimums, results that are an infinity or a NaN: the folds add s (c - 8) x and m x apart, which of an infinite x
// can leave NaN where (s (c - 8) + m) x is infinite, and the sum of 32 values close to fp32's largest can pass it.  Those are
// summed again term by term in 64 bits, of a row with infinities these alone; beside a NaN everything is one already.
// A wave for one row of x: what the row has in it ...
enum { ROW_FINITE = 0, ROW_INF = 1, ROW_NAN = 2 };
template <int DT> __device__ __forceinline__ int w4_kind(const W4Args & a, int row) {
    const typename Elem<DT>::T * x = static_cast<const typename Elem<DT>::T *>(a.x) + row * a.x_stride;
    bool inf = false, nan = false;
    for (int j = 8 * (threadIdx.x & 63); j < a.k; j += 512) {
        float t[8];
        load8<DT>(x + j, t);
#pragma unroll
        for (int i = 0; i < 8; i++) inf |= __builtin_fabsf(t[i]) == __builtin_inff(), nan |= t[i] != t[i];
    }
    return __ballot(nan) ? ROW_NAN : __ballot(inf) ? ROW_INF : ROW_FINITE;
}
// ... and its results, a column a lane
template <int DT> __device__ __forceinline__ float w4_terms(const W4Args & a, int row, int col, int kind) {
    const typename Elem<DT>::T * x = static_cast<const typename Elem<DT>::T *>(a.x) + row * a.x_stride;
    const uint8_t * cp = a.codes + (size_t) col * (a.k >> 1);
    const size_t s0 = (size_t) col * a.gs;
    double sum = 0;
#pragma unroll 1
    for (int j0 = 0; j0 < a.k; j0 += 512) {
        const int mine = j0 + 8 * (threadIdx.x & 63);
        bool look = mine < a.k;
        float t[8];
        if (look && kind == ROW_INF) {
            load8<DT>(x + mine, t);
            look = false;
#pragma unroll
            for (int i = 0; i < 8; i++) look |= __builtin_fabsf(t[i]) == __builtin_inff();
        }
#pragma unroll 1
        for (uint64_t todo = __ballot(look); todo; todo &= todo - 1) {
            const int j = j0 + 8 * (int) __builtin_ctzll(todo), g = j >> (5 + a.gsh);
            load8<DT>(x + j, t);
            const unsigned w = *reinterpret_cast<const unsigned *>(cp + (j >> 1));
            const double sc = h2f_bits(a.scales[s0 + g]), mn = h2f_bits(a.mins[s0 + g]);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (kind == ROW_FINITE || __builtin_fabsf(t[i]) == __builtin_inff())
                    sum += (sc * ((int) (w >> (8 * (i & 3) + (i & 4)) & 15u) - 8) + mn) * (double) t[i];
        }
        if (!__ballot(sum == sum)) break;
    }
    return (float) sum;
}
__device__ __forceinline__ bool wild(float v) { return !(__builtin_fabsf(v) < __builtin_inff()); }

// Those of a wave's own results, read back once all are stored.  Functions of their own, called where something is not finite: in
// line they changed the loops' schedules (64 rows of bf16 x 17,408 x 5,120: 92 -> 95 us, as calls 93).
__device__ __forceinline__ const W4Args * kernel_args() { return (const W4Args *) __builtin_amdgcn_kernarg_segment_ptr(); }
// k_w4: rows of x below MR, tiles of TR weight rows
template <int DT, int MR, int TR, int W>
__device__ __attribute__((noinline)) void w4_again(const W4Args * ap, int first, int step) {
    const W4Args a = *ap;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const bool one = a.wk_log == 0; // a wave per tile: its first TR lanes a column each; else the set's results over all threads
    const int wn = wave >> a.wk_log, WN = W >> a.wk_log, sets = ((a.n + TR - 1) / TR + WN - 1) / WN;
    const int i0 = one ? wn * MR * TR : wave * 64, i1 = one ? i0 + MR * TR : WN * MR * TR;
#pragma unroll 1
    for (int row = 0; row < min(MR, a.rows); row++) {
        int kind = -1;
#pragma unroll 1
        for (int set = first; set < sets && kind != ROW_NAN; set += step)
#pragma unroll 1
            for (int i = i0; i < i1; i += one ? TR : W * 64) {
                const int at = i + lane, col = (set * WN + at / TR / MR) * TR + at % TR;
                float * y = a.y + row * a.y_stride + col;
                const bool mine = at < i1 && (!one || lane < TR) && at / TR % MR == row && col < a.n && wild(*y);
                if (!__ballot(mine)) continue;
                if (kind < 0) kind = w4_kind<DT>(a, row);
                if (kind == ROW_NAN) break;
                const float v = w4_terms<DT>(a, row, mine ? col : 0, kind);
                if (mine) *y = v;
            }
    }
}
// k_w4_wide: 16 columns of four rows a wave
template <int DT, int TM, int NTW, int WN, int W>
__device__ __attribute__((noinline)) void w4_wide_again(const W4Args * ap, int t0, int t1, int row0) {
    const W4Args a = *ap;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
#pragma unroll 1
    for (int t = 0; t < NTW; t++)
#pragma unroll 1
        for (int i = wave * 64; i < WN * TM * 16; i += W * 64)
#pragma unroll 1
            for (int q = 0; q < 4; q++) {
                const int row = row0 + (i >> 4) % TM + q, tile = t0 + (i >> 4) / TM + WN * t, col = tile * 16 + n;
                float * y = a.y + row * a.y_stride + col;
                const bool mine = g == q && tile < t1 && col < a.n && row < a.rows && wild(*y);
                if (!__ballot(mine)) continue;
                const int kind = w4_kind<DT>(a, row);
                if (kind == ROW_NAN) continue;
                const float v = w4_terms<DT>(a, row, mine ? col : 0, kind);
                if (mine) *y = v;
            }
}

constexpr int W4_RUN = 2;   // steps a wave takes together: the 128 bytes of a cache line of every row (4 and 8: within 1% of it, with more code)
constexpr int W4_WIN = 32;  // scales of a weight row that a wave holds in LDS at a time
constexpr int W4_WROW = W4_WIN + 8; // ... a row's place: 16 rows' 80 bytes begin in different banks

// NR activation rows per group of four operand rows, RG groups: MR = NR RG rows a pass.
// What bounds it: the codes' way from HBM where there are many (150,001 x 5,120 on one row of units, group 32, 433 MB with x and y:
// 83 us, 5.2 TB/s of 6.0 that a plain read reaches; plain rows the codes' way to fp16, 52 of a step's 75 vector instructions: 84 to
// 87 us with group 128, 397 MB), else the chain of launch, x and first loads (1,024 x 5,120: 4.3 us).  Scalars do not all fit (23 to
// 70 of them are kept in lanes of vector registers), nor do the vector registers of fp32 rows with minimums (24 to 72 bytes of
// scratch a lane); neither is touched where the matrix instructions are.
// P parts: a tile is 16 / P weight rows, and lanes n = 16 / P h + j hold row j of part h, a P-th of its blocks.  A group's
// operand row NR h + m is then x[m] of part h's block (P NR <= 4), and a lane takes its own part's sums: with few
// rows of x the tiles get smaller, and a short projection has enough of them for every CU.
// W waves: 1 << wk_log of them share a tile, each a run of its steps, the others have tiles of their own.
// The codes of the next run are loaded while a run is worked on, over the tiles' borders too.  The scales come
// 32 a row at a time (64 contiguous bytes; a lane's own two bytes of each step would fetch every cache line many times),
// through LDS of the wave's own, in which every lane then finds its block's.
template <int MODE, int DT, int NR, int RG, int P, int W, bool MINS>
__global__ __launch_bounds__(W * 64, 4) void k_w4(W4Args a) {
    static_assert(P * NR <= 4, "parts share a group's four operand rows");
    constexpr int MR = NR * RG, BB = planes(MODE) * MR * 16, TR = 16 / P, U = W4_RUN;
    const W4Lds L = w4_lds<MODE, MR, MINS>(a.kcb);
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const float * dx = reinterpret_cast<const float *>(lds + L.dx), * ds = dx + a.kcb * MR;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int WK = 1 << a.wk_log, wk = wave & (WK - 1), wn = wave >> a.wk_log, WN = W >> a.wk_log;
    const int nb = a.k >> 5, tiles = (a.n + TR - 1) / TR, sets = (tiles + WN - 1) / WN;
    const int nbp = (nb + 4 * U * P - 1) / (4 * U * P) * (4 * U * P), pb = nbp / P; // blocks with padding, blocks of a part
    const int j = n % TR, h = n / TR;
    uint16_t * win = reinterpret_cast<uint16_t *>(lds + L.end) + wave * (MINS ? 2 : 1) * 16 * W4_WROW; // [16][40] scales, then m
    float * red = reinterpret_cast<float *>(lds + L.end + W * (MINS ? 2 : 1) * 16 * W4_WROW * 2);       // [2][waves][MR][TR]
    // the lane's piece of the diagonal operand: row n = 4 b + NR part + m, lane group b
    const int m = n % NR, a_part = (n & 3) / NR;
    const bool active = (n >> 2) == g && a_part < P;
    constexpr bool ROWS = MODE == XM_UNITS; // x by rows: a block's two units in its row's even or odd part
    const int abase = !active ? L.zero
                      : ROWS  ? m * L.row + (g & 1) * L.half + (a_part * pb + (g & 2)) * 16
                              : (a_part * pb + g) * BB + a_part * (pb / 8) * run_pad(MODE, MR) + m * 16;
    const int astep = !active ? 0 : ROWS ? 64 : 4 * BB, arun = U * astep + (!active || ROWS ? 0 : run_pad(MODE, MR)); // a step, a run
    const int agroup = !active ? 0 : ROWS ? NR * L.row : NR * 16;
    const int hb = P == 1 ? 0 : h * pb, myb = hb + g; // the first block of the lane's part, the lane's block of step 0
    // runs of the chunk of x that begins at block b0 (parts: all of x at once), and the wave's steps of them
    const auto runs = [&](int b0) { return (P == 1 ? min(a.kcb, nbp - b0) : pb) / (4 * U); };
    const auto begin = [&](int b0) { return U * ((runs(b0) * wk) >> a.wk_log); };
    const auto end = [&](int b0) { return U * ((runs(b0) * (wk + 1)) >> a.wk_log); };
    // what the wave loads next: a tile's first row in scalars, the lane's row and block in 32 bits
    struct Next {
        int set, b0, s, sw; // sw: the step at which the window of scales begins
        const uint8_t * cp;
        const uint16_t * sp, * mp;
        unsigned vc, vs;
    } nx;
    const int G = gridDim.x, wsteps = (W4_WIN / 4) << a.gsh;
    bool fresh = false; // nx begins a window: its scales (and m) are in the registers below
    u32x4 ws, wm;
    const auto window = [&] {
        nx.sw = nx.s;
        fresh = true;
        const int first = (hb + nx.b0 + 4 * nx.s) >> a.gsh; // (exact: runs and parts are whole groups)
        // (only what the wave's steps of this window need: 8 g groups in)
        if (8 * g < (4 * (end(nx.b0) - nx.s) + 3) >> a.gsh) {
            ws = w4_scales(nx.sp + nx.vs, a.gs, first + 8 * g);
            if constexpr (MINS) wm = w4_scales(nx.mp + nx.vs, a.gs, first + 8 * g);
        }
    };
    const auto enter = [&](int set) {
        const int first = min((set * WN + wn) * TR, a.n - 1), nr = min(j, a.n - 1 - first);
        nx.set = set;
        nx.b0 = 0;
        nx.s = begin(0);
        nx.cp = a.codes + (size_t) first * (a.k >> 1);
        nx.sp = a.scales + (size_t) first * a.gs;
        nx.mp = a.mins + (size_t) first * a.gs;
        nx.vc = (unsigned) (nr * (a.k >> 1));
        nx.vs = (unsigned) (nr * a.gs);
    };
    const auto load = [&](int u) {
        const unsigned blk = (unsigned) min(nx.b0 + 4 * (nx.s + u) + myb, nb - 1); // (past the last block the factors of x are zero)
        return *reinterpret_cast<const u32x4 *>(nx.cp + (nx.vc + blk * 16));
    };
    const auto advance = [&] { // (past the launch's last run: that run once more, unused)
        fresh = false;
        nx.s += U;
        if (nx.s < end(nx.b0)) {
            if (nx.s - nx.sw >= wsteps) window();
            return;
        }
        int b0 = nx.b0, s;
        do {
            b0 += P == 1 ? a.kcb : nbp;
            s = begin(b0);
        } while (b0 < nbp && s >= end(b0)); // (a last chunk without a run of this wave's)
        if (b0 < nbp) {
            nx.b0 = b0;
            nx.s = s;
            window();
        } else if (nx.set + G < sets) {
            enter(nx.set + G);
            window();
        } else nx.s -= U;
    };
    constexpr bool TERMS = MINS && MODE != XM_UNITS; // results that are not finite are looked at again
    bool again = false;
    enter(blockIdx.x);
    window();
    u32x4 in[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        in[u] = load(u);
        __builtin_amdgcn_sched_barrier(0); // (in the loop's order: its waits count the younger loads)
    }
    float acc[RG][NR];
    int par = 0, sw = 0;
    bool staged = false;
    for (int set = blockIdx.x; set < sets; set += G, par ^= 1) {
#pragma unroll
        for (int i = 0; i < RG; i++)
#pragma unroll
            for (int r = 0; r < NR; r++) acc[i][r] = 0.f;
        for (int b0 = 0; b0 < nbp; b0 += P == 1 ? a.kcb : nbp) {
            if (!staged) {
                __syncthreads();
                w4_stage<MODE, DT, MR, W, MINS>(a, lds, b0, P == 1 ? min(a.kcb, nbp - b0) : nbp);
                __syncthreads();
                staged = nbp <= a.kcb;
            }
            const int s1 = end(b0);
            int ax = abase + begin(b0) / U * arun;
#pragma unroll 1
            for (int s = begin(b0); s < s1; s += U, ax += arun) {
                if (fresh) { // (the run's window: nx stands on this run)
                    *reinterpret_cast<u32x4 *>(win + n * W4_WROW + 8 * g) = ws;
                    if constexpr (MINS) *reinterpret_cast<u32x4 *>(win + (16 + n) * W4_WROW + 8 * g) = wm;
                    asm volatile("" ::: "memory"); // (read below by other lanes and as another type)
                    sw = s;
                }
                advance();
                const uint16_t * wp = win + n * W4_WROW;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    // the codes leave their registers, then the next run's take them
                    const int at = (4 * (s + u - sw) + g) >> a.gsh;
                    const float sc = h2f_bits(wp[at]), mn = MINS ? h2f_bits(wp[16 * W4_WROW + at]) : 0.f;
                    i32x4 hbv[2];
                    half8 hw[4];
                    if constexpr (MODE == XM_UNITS) {
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            int t0, t1;
                            w4_bytes(in[u][k], t0, t1);
                            hbv[k >> 1][2 * (k & 1)] = t0;
                            hbv[k >> 1][2 * (k & 1) + 1] = t1;
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; k++) hw[k] = w4_halves(in[u][k]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    in[u] = load(u);
                    __builtin_amdgcn_sched_barrier(0);
                    const uint8_t * ap = lds + (ax + u * astep);
                    const float * dxp = dx + (4 * (s + u) + myb) * MR, * dsp = ds + (4 * (s + u) + myb) * MR;
                    // the sums of the lane's own part
                    const auto mine = [&](const auto & c, int r) {
                        if constexpr (P == 1) return c[r];
                        else if constexpr (P == 2) return h ? c[NR + r] : c[r];
                        else return h & 2 ? (h & 1 ? c[3] : c[2]) : (h & 1 ? c[1] : c[0]);
                    };
#pragma unroll
                    for (int i = 0; i < RG; i++) {
                        if constexpr (MODE == XM_UNITS) {
                            const i32x4 a0 = *reinterpret_cast<const i32x4 *>(ap + i * agroup), a1 = *reinterpret_cast<const i32x4 *>(ap + i * agroup + 16);
                            i32x4 c = {0, 0, 0, 0};
                            c = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, hbv[0], c, 0, 0, 0);
                            c = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, hbv[1], c, 0, 0, 0);
#pragma unroll
                            for (int r = 0; r < NR; r++) acc[i][r] = __builtin_fmaf((float) mine(c, r), sc * dxp[NR * i + r], acc[i][r]);
                        } else {
                            f32x4 c = {0, 0, 0, 0};
#pragma unroll
                            for (int k = planes(MODE) - 1; k >= 0; k--)
                                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const half8 *>(ap + (k * MR + i * NR) * 16), hw[k & 3], c, 0, 0, 0);
#pragma unroll
                            for (int r = 0; r < NR; r++) acc[i][r] = __builtin_fmaf(mine(c, r), sc * dxp[NR * i + r], acc[i][r]);
                        }
                        if constexpr (MINS) {
#pragma unroll
                            for (int r = 0; r < NR; r++) acc[i][r] = __builtin_fmaf(mn, dsp[NR * i + r], acc[i][r]);
                        }
                    }
                }
            }
        }
        const int tile = set * WN + wn;
        // the four lane groups' blocks, the parts, then the waves of the tile in order
#pragma unroll
        for (int i = 0; i < RG; i++)
#pragma unroll
            for (int r = 0; r < NR; r++) {
                acc[i][r] = quad_sum(acc[i][r]);
                if constexpr (P >= 2) acc[i][r] += shfl_xor(acc[i][r], 8);
                if constexpr (P >= 4) acc[i][r] += shfl_xor(acc[i][r], 4);
            }
        if (WK == 1) {
            if (lane < TR && tile * TR + lane < a.n) {
#pragma unroll
                for (int i = 0; i < MR; i++)
                    if (i < a.rows) {
                        a.y[i * a.y_stride + tile * TR + lane] = acc[i / NR][i % NR];
                        if (TERMS) again |= wild(acc[i / NR][i % NR]);
                    }
            }
            continue;
        }
        float * rp = red + par * (W * MR * TR);
        if (lane < TR) {
#pragma unroll
            for (int i = 0; i < MR; i++) rp[(wave * MR + i) * TR + lane] = acc[i / NR][i % NR];
        }
        __syncthreads(); // (the other parity's sums are not written again before every wave has passed this barrier)
        for (int i = threadIdx.x; i < WN * MR * TR; i += W * 64) {
            const int c = i % TR, mm = i / TR % MR, t = i / TR / MR, col = (set * WN + t) * TR + c;
            float v = rp[((t << a.wk_log) * MR + mm) * TR + c];
            for (int k = 1; k < WK; k++) v += rp[(((t << a.wk_log) + k) * MR + mm) * TR + c];
            if (col < a.n && mm < a.rows) {
                a.y[mm * a.y_stride + col] = v;
                if (TERMS) again |= wild(v);
            }
        }
    }
    if constexpr (TERMS) {
        if (__builtin_expect(__ballot(again) != 0, 0)) w4_again<DT, MR, TR, W>(kernel_args(), blockIdx.x, G);
    }
}

// ------------------------------------------------------------------------------------------------ more than 8 rows
// With more rows of x the diagonal operand's zeros cost: three of four lanes' LDS reads and matrix multiplications.  Here the
// four dwords of a block's codes go to the four lane groups instead (a 4 x 4 exchange of registers and lane groups), so
// that one instruction takes 16 rows of x against one block of 16 weight rows, without zeros, and every lane has its weight
// row's scale of each block.  A workgroup takes up to 2 NTW tiles: 4 waves along the blocks of a chunk (U steps each) times 2
// along the tiles; a piece of x read from LDS serves the wave's NTW tiles.  What bounds it is the fold of the blocks'
// integer sums into fp32, three instructions per (row, block, weight row) in three of four vector instructions (64 rows of
// 17,408 x 5,120: 35 us, the vector units busy for 74% of them, the matrix units for 16%).
__device__ __forceinline__ void w4_exchange(const u32x4 & d, unsigned (&t)[4]) { // t[b] in lane group q: dword q of lane group b's d
    const auto x = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false), y = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
    const auto v = __builtin_amdgcn_permlane16_swap(x[0], y[0], false, false), w = __builtin_amdgcn_permlane16_swap(x[1], y[1], false, false);
    t[0] = v[0], t[1] = v[1], t[2] = w[0], t[3] = w[1];
}

// LDS of a chunk of x, CB blocks of TM rows.  Units: a row's CB units of the even blocks, then CB of the odd ones (one 1 KiB
// copy brings 64 of them from two contiguous pieces of memory), 16 bytes of padding behind each copy (16 rows' pieces
// then lie in different banks), and the factors [CB][TM + 4].  Plain rows: w4_stage's layout.
template <int MODE, int MT, int CB, bool MINS> constexpr int wide_buf() {
    constexpr int TM = 16 * MT;
    return MODE == XM_UNITS ? CB * 2 * TM / 64 * 1040 + (MINS ? 2 : 1) * CB * (TM + 4) * 4 : w4_lds<MODE, TM, MINS>(CB).end;
}

// WK waves along the blocks of a chunk, U steps each, times WN along the tiles.  ODD: a workgroup of an odd number of tiles,
// whose second half of the waves has one less, with a loop body of its own (64 rows of 17,408 x 5,120, five tiles a workgroup:
// 35 us, with the sixth worked on and dropped 41)
template <int MODE, int DT, int MT, int NTW, int WK, int WN, int U, bool ODD, bool MINS>
__global__ __launch_bounds__(WK * WN * 64, WK * WN / 4) void k_w4_wide(W4Args a) {
    constexpr int WIDE_W = WK * WN, TM = 16 * MT, CB = 4 * WK * U, BB = planes(MODE) * TM * 16, BUF = wide_buf<MODE, MT, CB, MINS>();
    // x copied into the other buffer while a chunk is worked on (its matrix instructions and folds: the compiler's waits for the chunk's
    // codes do not know of the copies issued behind them, so the exchange of the codes begins when most copies have landed)
    constexpr bool ASYNC = MODE == XM_UNITS;
    constexpr int RPC = 32 / CB; // rows of a copy
    constexpr int DX = ASYNC ? TM / RPC * 1040 : w4_lds<MODE, TM, MINS>(CB).dx, DS = ASYNC ? TM + 4 : TM; // the factors of x behind the blocks, their stride
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wk = wave % WK, wn = wave / WK;
    const int nb = a.k >> 5, tiles = (a.n + 15) >> 4, row0 = blockIdx.y * TM;
    const int t0 = blockIdx.x * a.kcb, t1 = min(tiles, t0 + a.kcb); // (kcb: tiles of a workgroup)
    const int chunks = (nb + CB - 1) / CB;

    // ---- x
    const unsigned base = (unsigned) __builtin_amdgcn_readfirstlane((unsigned) (size_t) (__attribute__((address_space(3))) uint8_t *) lds);
    constexpr int PAIRS = CB / 2 * TM, META = (PAIRS + WIDE_W * 64 - 1) / (WIDE_W * 64); // pairs of blocks whose scales a thread brings
    uint4 meta[META];
    const auto issue = [&](int c, int buf) { // units of chunk c on their way to LDS, their scales and sums to registers
        const int b0 = c * CB, part = lane / CB & 1, unit = min(b0 + lane % CB, nb - 1);
        const int8_t * src = part ? a.xb : a.xa;
#pragma unroll 1
        for (int k0 = wave; k0 < TM / RPC; k0 += WIDE_W) {
            const int k = (k0 + blockIdx.x) % (TM / RPC); // (every workgroup reads the same rows: each begins with others)
            const int row = min(row0 + k * RPC + lane / (2 * CB), a.rows - 1);
            dma16(src + ((size_t) row * nb + unit) * 16, base + buf * BUF + k * 1040);
        }
#pragma unroll
        for (int k = 0; k < META; k++) {
            const int i = min(tid + k * WIDE_W * 64, PAIRS - 1), m = i / (CB / 2), blk = min(b0 + i % (CB / 2) * 2, nb - 2), row = min(row0 + m, a.rows - 1);
            const uint2 * mp = reinterpret_cast<const uint2 *>(a.xmeta) + (size_t) row * nb + blk;
            const uint2 u0 = mp[0], u1 = mp[1];
            meta[k] = make_uint4(u0.x, u0.y, u1.x, u1.y);
        }
    };
    const auto commit = [&](int c, int buf) { // the factors of chunk c, zeros past the last block
        float * dx = reinterpret_cast<float *>(lds + buf * BUF + DX), * ds = dx + CB * DS;
#pragma unroll
        for (int k = 0; k < META; k++) {
            const int i = tid + k * WIDE_W * 64, m = i / (CB / 2), bl = i % (CB / 2) * 2;
            if (i >= PAIRS) continue;
            const uint4 v = meta[k];
            const bool in = c * CB + bl < nb;
            const float da = in ? h2f_bits((uint16_t) v.x) : 0.f, db = in ? h2f_bits((uint16_t) (v.x >> 16)) : 0.f;
            dx[bl * DS + m] = da * 0.0625f;
            dx[(bl + 1) * DS + m] = db * 0.0625f;
            if constexpr (MINS) {
                ds[bl * DS + m] = in ? da * (float) ((int) (int16_t) v.y + (int) (int16_t) v.w) : 0.f;
                ds[(bl + 1) * DS + m] = in ? db * (float) (((int) v.y >> 16) + ((int) v.w >> 16)) : 0.f;
            }
        }
    };

    // ---- weights: per tile the codes of the wave's U steps of a chunk, and its scales
    const uint8_t * cp[NTW];
    const uint16_t * sp[NTW], * mp[NTW];
#pragma unroll
    for (int t = 0; t < NTW; t++) {
        const int tile = t0 + wn + WN * t, row = min((tile < t1 ? tile : t0) * 16 + n, a.n - 1);
        cp[t] = a.codes + (size_t) row * (a.k >> 1);
        sp[t] = a.scales + (size_t) row * a.gs;
        mp[t] = MINS ? a.mins + (size_t) row * a.gs : nullptr;
    }
    const bool last = t0 + wn + WN * (NTW - 1) < t1;
    u32x4 in[NTW][U];
    u32x4 is[NTW], im[NTW];
    const auto load = [&](int c, int t, int u) {
        in[t][u] = *reinterpret_cast<const u32x4 *>(cp[t] + 16 * min(c * CB + 4 * (wk * U + u) + g, nb - 1));
    };
    const auto load_s = [&](int c, int t) {
        const int grp = (c * CB + 4 * wk * U) >> a.gsh;
        is[t] = w4_scales(sp[t], a.gs, grp);
        if constexpr (MINS) im[t] = w4_scales(mp[t], a.gs, grp);
    };

    // the scale of each block of the wave's steps from the groups'
    const auto blocks_of = [&](u32x4 e, float (&f)[4 * U]) {
        const auto lo = [](unsigned x) { return (x & 0xffffu) | x << 16; };
        const auto hi = [](unsigned x) { return (x & 0xffff0000u) | x >> 16; };
        if (a.gsh == 1) e = u32x4{lo(e[0]), hi(e[0]), lo(e[1]), hi(e[1])};
        else if (a.gsh == 2) e = u32x4{lo(e[0]), lo(e[0]), hi(e[0]), hi(e[0])};
#pragma unroll
        for (int k = 0; k < 4 * U; k++) f[k] = (float) as_h2(e[k >> 1])[k & 1];
    };
    float acc[NTW][MT][4];
#pragma unroll
    for (int t = 0; t < NTW; t++)
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[t][i][r] = 0.f;
    if constexpr (ASYNC) issue(0, 0);
#pragma unroll
    for (int t = 0; t < NTW; t++) {
#pragma unroll
        for (int u = 0; u < U; u++) load(0, t, u);
        load_s(0, t);
    }
    if constexpr (ASYNC) {
        commit(0, 0);
        vm_drain();
        __syncthreads();
    }
#pragma unroll 1
    for (int c = 0; c < chunks; c++) {
        const int buf = ASYNC ? c & 1 : 0, cn = min(c + 1, chunks - 1);
        if constexpr (ASYNC) issue(cn, buf ^ 1); // (past the last chunk: that one once more, unused)
        else {
            constexpr int NX = CB * 4 * TM / (WIDE_W * 64);
            W4Eighth<DT> xr[NX]; // (loaded a chunk ahead they would cost the second workgroup of a CU: 32 rows of 65,536 x 5,120 fp32, 115 us, then 165)
#pragma unroll
            for (int u = 0; u < NX; u++) xr[u].load(a, tid + u * WIDE_W * 64, TM, row0, c * CB);
            __syncthreads();
#pragma unroll
            for (int u = 0; u < NX; u++) xr[u].template store<MODE, TM, MINS>(a, lds, w4_lds<MODE, TM, MINS>(CB), tid + u * WIDE_W * 64, row0, c * CB);
            __syncthreads();
        }
        // the codes to their lane groups, the scales of each block to floats; the next chunk's take their registers
        unsigned bt[NTW][U][4];
        float sc[NTW][4 * U], mn[NTW][4 * U];
#pragma unroll
        for (int t = 0; t < NTW; t++) {
#pragma unroll
            for (int u = 0; u < U; u++) w4_exchange(in[t][u], bt[t][u]);
            blocks_of(is[t], sc[t]);
            if constexpr (MINS) blocks_of(im[t], mn[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < NTW; t++) {
            load_s(cn, t);
        }
#pragma unroll
        for (int t = 0; t < NTW; t++)
#pragma unroll
            for (int u = 0; u < U; u++) load(cn, t, u);
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t * xp = lds + buf * BUF;
        const float * dx = reinterpret_cast<const float *>(xp + DX), * ds = dx + CB * DS;
        const auto fold = [&](auto of) { // the wave's first `of` tiles
            constexpr int NT = decltype(of)::value;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int bl = 4 * (wk * U + u) + q;
                    i32x2 bi[NT];
                    half8 bh[NT];
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        if constexpr (MODE == XM_UNITS) {
                            int lo, hi;
                            w4_bytes(bt[t][u][q], lo, hi);
                            bi[t] = i32x2{lo, hi};
                        } else bh[t] = w4_halves(bt[t][u][q]);
                    }
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        // 16 rows of x and their factors, for every tile of the wave
                        f32x4 d = *reinterpret_cast<const f32x4 *>(dx + bl * DS + 16 * i + 4 * g), e;
                        if constexpr (MINS) e = *reinterpret_cast<const f32x4 *>(ds + bl * DS + 16 * i + 4 * g);
                        i32x2 xi;
                        if constexpr (MODE == XM_UNITS)
                            xi = *reinterpret_cast<const i32x2 *>(xp + (16 * i + n) / RPC * 1040 + (16 * i + n) % RPC * 512 + (bl & 1) * CB * 16 +
                                                                  (bl & ~1) * 16 + 8 * g);
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            f32x4 f;
                            if constexpr (MODE == XM_UNITS) {
                                i32x4 v = {0, 0, 0, 0};
                                v = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, xi), __builtin_bit_cast(long, bi[t]), v, 0, 0, 0);
#pragma unroll
                                for (int r = 0; r < 4; r++) f[r] = (float) v[r];
                            } else {
                                f = f32x4{0, 0, 0, 0};
#pragma unroll
                                for (int k = planes(MODE) - 4; k >= 0; k -= 4)
                                    f = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const half8 *>(xp + bl * BB + ((k + g) * TM + 16 * i + n) * 16),
                                                                               bh[t], f, 0, 0, 0);
                            }
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                acc[t][i][r] = __builtin_fmaf(f[r], sc[t][4 * u + q] * d[r], acc[t][i][r]);
                                if constexpr (MINS) acc[t][i][r] = __builtin_fmaf(mn[t][4 * u + q], e[r], acc[t][i][r]);
                            }
                        }
                    }
                    // (a block at a time: the compiler would fold the chunk's sums at its end, and they do not fit the registers)
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < MT; i++)
#pragma unroll
                            for (int r = 0; r < 4; r++) asm volatile("" : "+v"(acc[t][i][r]));
                }
        };
        if (!ODD || last) fold(std::integral_constant<int, NTW>{});
        else if constexpr (ODD) fold(std::integral_constant<int, NTW - 1>{});
        if constexpr (ASYNC) {
            commit(cn, buf ^ 1);
            // the copies of x have landed: the U codes of NTW tiles behind them may still be on their way
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NTW * U) : "memory");
            __syncthreads();
        }
    }
    constexpr bool TERMS = MINS && MODE != XM_UNITS;
    bool again = false;
    // the waves along the blocks, a tile of every wave at a time
    if constexpr (!ASYNC) __syncthreads();
    float * red = reinterpret_cast<float *>(lds); // [waves][TM][16]
#pragma unroll
    for (int t = 0; t < NTW; t++) {
        if (t) __syncthreads();
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) red[(wave * TM + 16 * i + 4 * g + r) * 16 + n] = acc[t][i][r];
        __syncthreads();
        for (int i = tid; i < WN * TM * 16; i += WIDE_W * 64) {
            const int c = i & 15, m = (i >> 4) % TM, w = (i >> 4) / TM, tile = t0 + w + WN * t, col = tile * 16 + c;
            const float * rp = red + (w * WK * TM + m) * 16 + c;
            float v = rp[0];
#pragma unroll
            for (int k = 1; k < WK; k++) v += rp[k * TM * 16];
            if (tile < t1 && col < a.n && row0 + m < a.rows) {
                a.y[(long long) (row0 + m) * a.y_stride + col] = v;
                if (TERMS) again |= wild(v);
            }
        }
    }
    if constexpr (TERMS) {
        if (__builtin_expect(__ballot(again) != 0, 0)) w4_wide_again<DT, TM, NTW, WN, WIDE_W>(kernel_args(), t0, t1, row0);
    }
}

constexpr int W4_LDS = 80 * 1024; // of k_w4: two workgroups per CU
constexpr int W4_WAVES = 4096; // of k_w4: 16 for each of 256 CUs

template <int MODE, int DT, int NR, int RG, int P, int W>
static hipError_t launch_k(W4Args a, hipStream_t st) {
    constexpr int MR = NR * RG, TR = 16 / P, PAD = 4 * W4_RUN;
    const int nb4 = (a.k / 32 + PAD * P - 1) / (PAD * P) * (PAD * P), tiles = (a.n + TR - 1) / TR;
    const int more = 2 * W * MR * TR * 4 + W * (a.mins ? 2 : 1) * 16 * W4_WROW * 2; // the waves' sums, the windows of scales
    const auto size = [&](int kcb) { return (a.mins ? w4_lds<MODE, MR, true>(kcb) : w4_lds<MODE, MR, false>(kcb)).end + more; };
    a.kcb = std::min(nb4, W4_LDS / (planes(MODE) * MR * 16 + MR * 4) / PAD * PAD);
    while (size(a.kcb) > W4_LDS) a.kcb -= PAD;
    if constexpr (P > 1) {
        if (a.kcb < nb4) return launch_k<MODE, DT, 4, (MR + 3) / 4, 1, 8>(a, st); // (x in pieces)
    }
    // (every wave has a run of the first chunk)
    while ((1 << a.wk_log) < W && (tiles << a.wk_log) < W4_WAVES / 2 && a.kcb / P / PAD >= 2 << a.wk_log) a.wk_log++;
    const int wn = W >> a.wk_log, sets = (tiles + wn - 1) / wn;
    const size_t lds = size(a.kcb);
    const dim3 grid(std::min(sets, W4_WAVES / W)), block(W * 64);
    static std::atomic<uint64_t> done[2];
    const auto k = a.mins ? k_w4<MODE, DT, NR, RG, P, W, true> : k_w4<MODE, DT, NR, RG, P, W, false>;
    const hipError_t e = allow_lds(k, lds, done[a.mins != nullptr]);
    if (e != hipSuccess) return e;
    return launch(k, grid, block, lds, st, a);
}

template <int MODE, int DT, int MT, int NTW, int WK, int WN, int U, bool ODD, bool MINS>
static hipError_t launch_wide_k(const W4Args & a, dim3 grid, hipStream_t st) {
    constexpr int WIDE_W = WK * WN;
    constexpr int lds = std::max((MODE == XM_UNITS ? 2 : 1) * wide_buf<MODE, MT, 4 * WK * U, MINS>(), WIDE_W * 16 * MT * 16 * 4);
    static_assert(lds <= 160 * 1024, "a workgroup's LDS");
    const auto k = k_w4_wide<MODE, DT, MT, NTW, WK, WN, U, ODD, MINS>;
    static std::atomic<uint64_t> done;
    const hipError_t e = allow_lds(k, lds, done);
    if (e != hipSuccess) return e;
    return launch(k, grid, dim3(WIDE_W * 64), lds, st, a);
}
template <int MODE, int DT, int MT, int U, bool MINS>
static hipError_t launch_wide_m(W4Args a, hipStream_t st) {
    // a workgroup per CU with up to 2 * 3 tiles each where that is all of them (16 rows of 17,408 x 5,120: 19 us, with two per
    // CU of four tiles 21), else two per CU with four tiles at a time, whose registers (and, of 64 rows, shorter chunks of x)
    // leave room for both (65,536: 16 rows 50 us, with rounds of 2 * 3 tiles 63; 64 rows 105 and 121)
    constexpr int CUS = 256, MOST = 6;
    const int tiles = (a.n + 15) / 16;
    const bool many = tiles > CUS * MOST;
    a.kcb = many ? 4 : (tiles + CUS - 1) / CUS;
    const dim3 grid((tiles + a.kcb - 1) / a.kcb, (a.rows + 16 * MT - 1) / (16 * MT));
    if (many) return launch_wide_k<MODE, DT, MT, 2, 4, 2, MT == 4 ? 1 : U, false, MINS>(a, grid, st);
    if constexpr (U == 2) { // one tile: all eight waves along the blocks
        if (a.kcb == 1) return launch_wide_k<MODE, DT, MT, 1, 8, 1, 1, false, MINS>(a, grid, st);
    }
    switch (a.kcb) {
    case 1:
    case 2: return launch_wide_k<MODE, DT, MT, 1, 4, 2, U, false, MINS>(a, grid, st);
    case 3: return launch_wide_k<MODE, DT, MT, 2, 4, 2, U, true, MINS>(a, grid, st);
    case 4: return launch_wide_k<MODE, DT, MT, 2, 4, 2, U, false, MINS>(a, grid, st);
    case 5: return launch_wide_k<MODE, DT, MT, 3, 4, 2, U, true, MINS>(a, grid, st);
    default: return launch_wide_k<MODE, DT, MT, 3, 4, 2, U, false, MINS>(a, grid, st);
    }
}
template <int MODE, int DT>
static hipError_t launch_wide(const W4Args & a, hipStream_t st) {
    if constexpr (MODE == XM_UNITS) {
        if (a.rows <= 16) return a.mins ? launch_wide_m<MODE, DT, 1, 2, true>(a, st) : launch_wide_m<MODE, DT, 1, 2, false>(a, st);
        if (a.rows <= 32) return a.mins ? launch_wide_m<MODE, DT, 2, 2, true>(a, st) : launch_wide_m<MODE, DT, 2, 2, false>(a, st);
        return a.mins ? launch_wide_m<MODE, DT, 4, 1, true>(a, st) : launch_wide_m<MODE, DT, 4, 2, false>(a, st);
    } else {
        if (a.rows <= 16) return a.mins ? launch_wide_m<MODE, DT, 1, 1, true>(a, st) : launch_wide_m<MODE, DT, 1, 1, false>(a, st);
        return a.mins ? launch_wide_m<MODE, DT, 2, 1, true>(a, st) : launch_wide_m<MODE, DT, 2, 1, false>(a, st);
    }
}

// By the rows of x, in us for 1,024 / 17,408 / 150,001 weight rows of 5,120, units, groups of 32:
//   1     four parts     4.6 / 13.2 / 82   whole tiles of 16 weight rows  6.4 / 15.9 / 92
//   2     two parts      5.3 / 13.7 / 87   whole tiles                    6.6 / 15.8 / 92
//   3, 4  one group      6.2 / 16.0 / 93   two groups                     7.4 / 17.4 / 95
//   5..8  two groups     7.2 / 17.5 / 97   dense                          7.2 / 18.4 / 118
//   16    dense          7.6 / 18.2 / 118  four groups                   19.7 / 25.5 / 137
template <int MODE, int DT>
static hipError_t launch_mode(const W4Args & a, hipStream_t st) {
    if (a.rows == 1) return launch_k<MODE, DT, 1, 1, 4, 4>(a, st);
    if (a.rows == 2) return launch_k<MODE, DT, 2, 1, 2, 4>(a, st);
    if (a.rows <= 4) return launch_k<MODE, DT, 4, 1, 1, 8>(a, st);
    if (a.rows <= 8) return launch_k<MODE, DT, 4, 2, 1, 8>(a, st);
    return launch_wide<MODE, DT>(a, st);
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
