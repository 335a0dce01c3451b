// Residual addition and root-mean-square norm of a row, with the normed row as int8 units (the activation form of the
// attention's output, kv_attn.hip) and / or as a row of the input's type.
//
//   h_j = round(x_j + r_j)                   (fp32 sum, rounded to the stream's type: what is stored is what is normed)
//   rs  = 1 / sqrt(sum_j h_j^2 / D + eps)    (64-bit sum, then rounded once to fp32)
//   y_j = (h_j rs) w_j
//   units, per block of 32: t_j = h_j w_j, a = max |t|, code = round_to_even(t_j (127 / a)), scale = fp16(a (rs / 127))
// The codes are taken before the norm's factor, which cancels in t / a: they then depend on nothing that a sum's order
// changes, and with the sum in 64 bits neither do rs and the scales.
// In a row whose rs = m 2^e is far from one (values near fp32's ends that eps does not lift) rs itself, t or 127 / a would leave
// fp32's range, or its normal numbers, where y does not: there h_j 2^e and m take the places of h_j and rs, with the same bits.
#include "step_dev.h"

namespace qkv {

constexpr int NORM_FAR = 32; // the largest |e| of a row that is worked on as it is
// a block whose largest value is below this has no finite 127 / a; with rs up to 2^32 its scale is far below 2^-25, zero in fp16,
// and so are its codes
constexpr float NORM_TINY = 4e-37f;

// A workgroup per row; thread t holds the chunks t, t + NT, .. (C of them) of 8 values, so a block of 32 is four
// neighbouring lanes.
template <int DT, int C>
__global__ __launch_bounds__(1024) void k_norm(NormArgs a) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ double red[16];
    const int tid = threadIdx.x, wave = tid >> 6, NT = blockDim.x;
    const int nu = a.dim >> 5;
    int j[C], n[C]; // the chunks' first values and how many of the 8 exist
#pragma unroll
    for (int c = 0; c < C; c++) {
        j[c] = 8 * (tid + NT * c);
        n[c] = max(0, min(8, a.dim - j[c]));
    }
    const int row = blockIdx.x;
    const T * xp = static_cast<const T *>(a.x) + (long long) row * a.x_stride;
    const T * rp = static_cast<const T *>(a.res) + (long long) row * a.res_stride;
    float h[C][8], r[C][8], w[C][8];
#pragma unroll
    for (int c = 0; c < C; c++) {
#pragma unroll
        for (int i = 0; i < 8; i++) h[c][i] = 0.f;
        if (n[c] <= 0) continue;
        load_n<DT>(xp + j[c], n[c], h[c]);
        if (a.res) load_n<DT>(rp + j[c], n[c], r[c]);
        load_n<DT_F32>(a.w + j[c], n[c], w[c]);
    }
    double s = 0;
    if (a.res) {
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) h[c][i] = n[c] > 0 ? E::up(E::down(h[c][i] + r[c][i])) : 0.f;
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
        if (a.sum && n[c] > 0) store_n<DT>(static_cast<T *>(a.sum) + (long long) row * a.sum_stride + j[c], n[c], h[c]);
#pragma unroll
        for (int i = 0; i < 8; i++) s = __builtin_fma((double) h[c][i], (double) h[c][i], s);
    }
    s = wave_sum(s);
    if ((tid & 63) == 0) red[wave] = s;
    lds_barrier();
    s = red[0];
    for (int i = 1; i < NT / 64; i++) s += red[i];
    double rs64 = 1.0 / __builtin_sqrt(s / a.dim + (double) a.eps);
    const int e = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_exp(rs64)); // (0 of zero, an infinity and a NaN)
    if (__builtin_expect(e < -NORM_FAR || e > NORM_FAR, 0)) {
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) h[c][i] = __builtin_ldexpf(h[c][i], e);
        rs64 = __builtin_ldexp(rs64, -e);
    }
    const float rs = (float) rs64;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int ch = tid + NT * c;
        if (n[c] <= 0) continue; // (units: dim is a multiple of 64, so whole blocks of four lanes leave)
        if (a.y) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = (h[c][i] * rs) * w[c][i];
            store_n<DT>(static_cast<T *>(a.y) + (long long) row * a.y_stride + j[c], n[c], y);
        }
        if (a.a) {
            float t[8], am = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                t[i] = h[c][i] * w[c][i];
                am = fmaxf(am, fabsf(t[i]));
            }
            am = fmaxf(am, shfl_xor(am, 1));
            am = fmaxf(am, shfl_xor(am, 2));
            const float id = am < NORM_TINY ? 0.f : 127.0f / am;
            int sum = 0;
            unsigned q[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int v = f2i_rn(t[i] * id);
                sum += v;
                q[i >> 2] |= ((unsigned) v & 0xffu) << (8 * (i & 3));
            }
            sum += (int) shfl_xor_u((unsigned) sum, 1); // the half of 16 values
            const unsigned sc = f2h_bits(am < NORM_TINY ? am * 0.f * rs : am * (rs / 127.0f));
            const int blk = ch >> 2, part = blk & 1, gi = 2 * (blk >> 1) + ((ch >> 1) & 1);
            const long long u = (long long) row * nu + gi;
            *reinterpret_cast<uint2 *>((part ? a.b : a.a) + u * 16 + 8 * (ch & 1)) = make_uint2(q[0], q[1]);
            // meta: scale of the even / odd block, sum of the even / odd half (the odd block is four lanes away)
            const unsigned mine = sc | (unsigned) sum << 16, other = shfl_xor_u(mine, 4);
            if (!(ch & 5))
                *reinterpret_cast<uint2 *>(a.meta + u * 4) = make_uint2((mine & 0xffffu) | other << 16, mine >> 16 | (other & 0xffff0000u));
        }
    }
}

// Chunks per thread: one for few rows, whose time is the row's chain of load, sum and store (1 row of 5,120: 3.5 us, with
// four 5.2; 32 rows 4.7 and 7.0), two for many, which leave room for more rows per CU (4,096 rows of bf16, residual and units:
// 37 us or 4.0 TB/s of what has to move, with one 40, with four 44; persistent workgroups that read the next row ahead 47 to
// 62: their registers leave half the waves), four only where two are not enough for 1,024 threads.
constexpr int NORM_FEW = 512;
template <int DT>
static hipError_t launch_dt(const NormArgs & a, hipStream_t st) {
    const int chunks = (a.dim + 7) / 8;
    const auto nt = [&](int c) { return dim3((chunks + 64 * c - 1) / (64 * c) * 64); };
    if (chunks <= 1024 && a.rows <= NORM_FEW) return launch(k_norm<DT, 1>, dim3(a.rows), nt(1), 0, st, a);
    if (chunks <= 2048) return launch(k_norm<DT, 2>, dim3(a.rows), nt(2), 0, st, a);
    return launch(k_norm<DT, 4>, dim3(a.rows), nt(4), 0, st, a);
}

hipError_t launch_norm(const NormArgs & a, int dtype, hipStream_t st) {
    return dtype == DT_F32 ? launch_dt<DT_F32>(a, st) : dtype == DT_F16 ? launch_dt<DT_F16>(a, st) : launch_dt<DT_BF16>(a, st);
}

} // namespace qkv
