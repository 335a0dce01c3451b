// Verification of drafted tokens against the target's distribution, from given random numbers.
//
//   p_i = softmax(logits_i / T) (or the probabilities given); draft d_i is accepted while u_i q_i(d_i) < p_i(d_i), q_i the
//   draft model's probabilities, or all on d_i without one.  At the first refusal i the next token is drawn from
//   max(p_i - q_i, 0), after the last draft from p_n: the first index at which the cumulative sum of the weights exceeds
//   u_n times their total (a random number of its own: the u_i that refused a draft is not free any more).
//
// A border of the cumulative sum lies near every random number when a vocabulary's 150,000 weights are small, so weights,
// sums and the comparison are in 64 bits: two orders of summation then differ by 1e-16 of the total, and a token changes
// with a probability of 1e-11.
//
// k_verify_rows: every row once, in slices of 4,096 entries (the slice's largest logit and its sum relative to that).
// k_verify_residual (with q): the slices' sums of max(p - q, 0) of the one row that was refused, if any.
// k_verify_pick: one workgroup per sequence: the decision, the slice of the next token by the slices' sums, and the token
// inside the slice.
#include "step_dev.h"

namespace qkv {

constexpr int VT = 256;      // threads
constexpr int VE = VERIFY_SLICE / VT; // entries per thread

constexpr double ln2_pow(int k) { // ln(2)^k / k!
    double c = 1;
    for (int i = 1; i <= k; i++) c *= 0.693147180559945309417232 / i;
    return c;
}
// 2^y for y <= 0 (NaN and far below: 0): y = n + f with |f| <= 1/2, the Taylor series of 2^f to the 11th power (the rest is
// below (ln(2) / 2)^12 / 12! = 6e-15 of it)
__device__ __forceinline__ double exp2_neg(double y) {
    y = __builtin_fmax(y, -2000.0);
    const double n = __builtin_rint(y), f = y - n;
    double p = ln2_pow(11);
#pragma unroll
    for (int k = 10; k >= 0; k--) {
        constexpr double c[11] = {ln2_pow(0), ln2_pow(1), ln2_pow(2), ln2_pow(3), ln2_pow(4), ln2_pow(5), ln2_pow(6), ln2_pow(7), ln2_pow(8), ln2_pow(9), ln2_pow(10)};
        p = __builtin_fma(p, f, c[k]);
    }
    return __builtin_ldexp(p, (int) n);
}

// a sequence's temperature: beta = log2(e) / T, 0 for greedy
struct Temp {
    double beta;
    bool greedy;
};
__device__ __forceinline__ Temp temp_of(const VerifyArgs & a, int b) {
    const float t = a.temp ? a.temp[b] : 1.f;
    const bool greedy = !(t > 0.f);
    return Temp{greedy ? 0.0 : 1.4426950408889634073599 / (double) t, greedy};
}
__device__ __forceinline__ int count_of(const VerifyArgs & a, int b) { return a.n_drafts ? max(0, min(a.n_drafts[b], a.n)) : a.n; }

template <bool PROBS> __device__ __forceinline__ double weight(float v, float top, double beta) {
    if constexpr (PROBS) return v > 0.f ? (double) v : 0.0;
    else return exp2_neg(((double) v - (double) top) * beta);
}

// 16 consecutive entries of a row from j on; those past the end are -infinity / 0
template <int DT> __device__ __forceinline__ void load16(const typename Elem<DT>::T * p, int j, int vocab, float none, float (&v)[VE]) {
#pragma unroll
    for (int c = 0; c < VE; c += 8) {
        float t[8];
        const int n = vocab - (j + c);
        if (n > 0) load_n<DT>(p + j + c, n, t);
#pragma unroll
        for (int i = 0; i < 8; i++) v[c + i] = i < n ? t[i] : none;
    }
}

template <int DT, bool PROBS>
__global__ __launch_bounds__(VT) void k_verify_rows(VerifyArgs a) {
    __shared__ float top[VT / 64];
    __shared__ double sums[VT / 64];
    __shared__ int args[VT / 64], bad[VT / 64];
    const int row = blockIdx.x / a.nsl, sl = blockIdx.x - row * a.nsl, b = row / (a.n + 1), i = row - b * (a.n + 1);
    if (i > count_of(a, b)) return; // (a row behind the sequence's last draft)
    const Temp t = temp_of(a, b);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, j0 = sl * VERIFY_SLICE + threadIdx.x * VE;
    float v[VE];
    load16<DT>(static_cast<const typename Elem<DT>::T *>(a.target) + (long long) row * a.row_stride, j0, a.vocab, PROBS ? 0.f : -__builtin_inff(), v);
    float m = -__builtin_inff();
    bool wild = false;
#pragma unroll
    for (int k = 0; k < VE; k++) {
        wild |= !(v[k] < __builtin_inff()); // +infinity or NaN
        m = fmaxf(m, v[k]);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, shfl_xor(m, x));
    if (lane == 0) top[wave] = m;
    const uint64_t any = __ballot(wild);
    if (lane == 0) bad[wave] = any != 0;
    __syncthreads();
    wild = false;
#pragma unroll
    for (int k = 0; k < VT / 64; k++) {
        m = fmaxf(m, top[k]);
        wild |= bad[k] != 0;
    }
    VerifyPart p{0.0, PROBS ? 0.f : m, 0};
    if (wild) p.top = __builtin_nanf("");
    else if (!PROBS && t.greedy) {
        int arg = 0x7fffffff;
#pragma unroll
        for (int k = VE - 1; k >= 0; k--) arg = v[k] == m && j0 + k < a.vocab ? j0 + k : arg;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) arg = min(arg, (int) shfl_xor_u((unsigned) arg, x));
        if (lane == 0) args[wave] = arg;
        __syncthreads();
        p.arg = args[0];
#pragma unroll
        for (int k = 1; k < VT / 64; k++) p.arg = min(p.arg, args[k]);
        p.sum = m > -__builtin_inff() ? 1.0 : 0.0;
    } else {
        double s = 0;
        if (PROBS || m > -__builtin_inff()) {
#pragma unroll
            for (int k = 0; k < VE; k++) s += weight<PROBS>(v[k], m, t.beta);
        }
        s = wave_sum(s);
        if (lane == 0) sums[wave] = s;
        __syncthreads();
        p.sum = sums[0];
#pragma unroll
        for (int k = 1; k < VT / 64; k++) p.sum += sums[k];
    }
    if (threadIdx.x == 0) a.part[(size_t) row * a.nsl + sl] = p;
}

// what every workgroup of a sequence finds from the slices' sums
struct Verdict {
    float top[VERIFY_MAX_DRAFTS + 1];  // per row: the largest logit
    double z[VERIFY_MAX_DRAFTS + 1];   // the sum of the weights relative to it (probabilities: their sum); not > 0: no row
    int arg[VERIFY_MAX_DRAFTS + 1];
    int acc;
};

// all VT threads; draws the accepted count and, when p is given, stores the drafts' probabilities
template <int DT, bool PROBS>
__device__ __forceinline__ void decide(const VerifyArgs & a, int b, int count, const Temp t, Verdict & V, float * p) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float ninf = -__builtin_inff();
    for (int i = wave; i <= count; i += VT / 64) {
        const VerifyPart * pp = a.part + (size_t) (b * (a.n + 1) + i) * a.nsl;
        float m = ninf;
        bool wild = false;
        for (int s = lane; s < a.nsl; s += 64) {
            const float x = pp[s].top;
            wild |= x != x;
            m = fmaxf(m, x);
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, shfl_xor(m, x));
        wild = __ballot(wild) != 0;
        double z = 0;
        int arg = 0x7fffffff;
        for (int s = lane; s < a.nsl; s += 64) {
            const VerifyPart x = pp[s];
            if (!PROBS && t.greedy) {
                if (x.top == m) arg = min(arg, x.arg);
            } else if (x.sum > 0) z += PROBS ? x.sum : x.sum * exp2_neg(((double) x.top - (double) m) * t.beta);
        }
        if (!PROBS && t.greedy) {
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) arg = min(arg, (int) shfl_xor_u((unsigned) arg, x));
            z = m > ninf ? 1.0 : 0.0;
        } else z = wave_sum(z);
        if (lane == 0) {
            V.top[i] = m;
            V.z[i] = wild || !(z < (double) __builtin_inff()) ? 0.0 : z;
            V.arg[i] = arg;
        }
    }
    __syncthreads();
    if (wave == 0) { // a draft per lane
        double pd = 0;
        bool ok = false;
        if (lane < count) {
            const int d = a.drafts[b * a.n + lane];
            const double z = V.z[lane];
            if (d >= 0 && d < a.vocab && z > 0) {
                if (!PROBS && t.greedy) pd = d == V.arg[lane] ? 1.0 : 0.0;
                else {
                    const float v = Elem<DT>::up(static_cast<const typename Elem<DT>::T *>(a.target)[(long long) (b * (a.n + 1) + lane) * a.row_stride + d]);
                    pd = weight<PROBS>(v, V.top[lane], t.beta);
                    if (!PROBS) pd /= z;
                }
                const double qd = a.q ? (double) a.q[((size_t) b * a.n + lane) * a.vocab + d] : 1.0;
                ok = (double) a.u[b * (a.n + 1) + lane] * qd < pd;
            }
        }
        const uint64_t no = ~__ballot(ok);
        if (lane == 0) V.acc = min(count, no ? (int) __builtin_ctzll(no) : 64);
        if (p && lane < a.n) p[b * a.n + lane] = (float) pd;
    }
    __syncthreads();
}

// the weights of 16 entries of the row the next token is drawn from
struct Source {
    long long row;   // of the target
    const float * q; // subtracted, or null
    float top;
    double beta, zinv;
    int skip;        // an entry that counts as zero (-1: none)
};
template <int DT, bool PROBS>
__device__ __forceinline__ void weights16(const VerifyArgs & a, const Source & S, int j, double (&w)[VE]) {
    float v[VE];
    load16<DT>(static_cast<const typename Elem<DT>::T *>(a.target) + S.row * a.row_stride, j, a.vocab, PROBS ? 0.f : -__builtin_inff(), v);
#pragma unroll
    for (int k = 0; k < VE; k++) w[k] = j + k == S.skip ? 0.0 : weight<PROBS>(v[k], S.top, S.beta);
    if (S.q) {
        float q[VE];
        load16<DT_F32>(S.q, j, a.vocab, 0.f, q);
#pragma unroll
        for (int k = 0; k < VE; k++) {
            const double r = (PROBS ? w[k] : w[k] * S.zinv) - (double) q[k];
            w[k] = r > 0 ? r : 0.0;
        }
    }
}

template <int DT, bool PROBS>
__global__ __launch_bounds__(VT) void k_verify_residual(VerifyArgs a) {
    __shared__ Verdict V;
    __shared__ double sums[VT / 64];
    const int b = blockIdx.x / a.nsl, sl = blockIdx.x - b * a.nsl, count = count_of(a, b);
    const Temp t = temp_of(a, b);
    if (!PROBS && t.greedy) return;
    decide<DT, PROBS>(a, b, count, t, V, nullptr);
    const int r = V.acc;
    if (r == count || !(V.z[r] > 0)) return;
    const Source S{(long long) b * (a.n + 1) + r, a.q + ((size_t) b * a.n + r) * a.vocab, V.top[r], t.beta, 1.0 / V.z[r], -1};
    double w[VE], s = 0;
    weights16<DT, PROBS>(a, S, sl * VERIFY_SLICE + threadIdx.x * VE, w);
#pragma unroll
    for (int k = 0; k < VE; k++) s += w[k];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = sums[0];
        for (int k = 1; k < VT / 64; k++) s += sums[k];
        a.rest[(size_t) b * a.nsl + sl] = s;
    }
}

// exclusive sum over the VT threads' values, and the total: thread k + 1's sum is thread k's sum plus its value
__device__ __forceinline__ double block_scan(double v, double * tmp, double & total) {
    tmp[threadIdx.x] = v;
    __syncthreads();
    double ex = 0, all = 0;
    for (int k = 0; k < VT; k++) {
        if (k == (int) threadIdx.x) ex = all;
        all += tmp[k];
    }
    total = all;
    __syncthreads();
    return ex;
}

template <int DT, bool PROBS>
__global__ __launch_bounds__(VT) void k_verify_pick(VerifyArgs a) {
    __shared__ Verdict V;
    __shared__ double tmp[VT], s_base;
    __shared__ int s_at, s_last;
    const int b = blockIdx.x, count = count_of(a, b), tid = threadIdx.x;
    const Temp t = temp_of(a, b);
    decide<DT, PROBS>(a, b, count, t, V, a.p);
    const int r = V.acc;
    int token = -1;
    if (V.z[r] > 0) {
        if (!PROBS && t.greedy) token = V.arg[r];
        else {
            const long long row = (long long) b * (a.n + 1) + r;
            const VerifyPart * pp = a.part + row * a.nsl;
            const bool refused = r < count;
            Source S{row, nullptr, V.top[r], t.beta, 1.0 / V.z[r], -1};
            if (refused) {
                if (a.q) S.q = a.q + ((size_t) b * a.n + r) * a.vocab;
                else {
                    const int d = a.drafts[b * a.n + r];
                    if (d >= 0 && d < a.vocab) S.skip = d;
                }
            }
            const int per = (a.nsl + VT - 1) / VT; // slices per thread
            const double u = (double) a.u[b * (a.n + 1) + a.n];
            for (int pass = 0; pass < 2; pass++) { // (again without q and skip where they leave nothing)
                // the sum of the skipped entry's slice, without it
                double less = 0;
                if (S.skip >= 0) {
                    double w[VE], s = 0;
                    weights16<DT, PROBS>(a, S, S.skip / VERIFY_SLICE * VERIFY_SLICE + tid * VE, w);
#pragma unroll
                    for (int k = 0; k < VE; k++) s += w[k];
                    (void) block_scan(s, tmp, less);
                }
                const auto slice = [&](int s) -> double {
                    if (s >= a.nsl) return 0.0;
                    if (S.q) return a.rest[(size_t) b * a.nsl + s];
                    if (S.skip >= 0 && s == S.skip / VERIFY_SLICE) return less;
                    const double x = pp[s].sum;
                    return PROBS ? x : x > 0 ? x * exp2_neg(((double) pp[s].top - (double) S.top) * S.beta) : 0.0;
                };
                double mine = 0, total;
                for (int k = 0; k < per; k++) mine += slice(tid * per + k);
                const double ex = block_scan(mine, tmp, total);
                if (!(total > 0)) {
                    S.q = nullptr;
                    S.skip = -1;
                    continue;
                }
                if (tid == 0) s_at = s_last = -1;
                __syncthreads();
                const double want = u * total;
                if (mine > 0) {
                    const bool here = ex <= want && want < ex + mine;
                    double run = ex;
                    int last = -1;
                    for (int k = 0; k < per; k++) {
                        const double x = slice(tid * per + k);
                        if (!(x > 0)) continue;
                        last = tid * per + k;
                        if (here) {
                            s_at = last;
                            s_base = run;
                            run += x;
                            if (want < run) break;
                        }
                    }
                    atomicMax(&s_last, last);
                }
                __syncthreads();
                // (want at or past the total, for a random number of 1 or more: the last slice with a weight, its last entry)
                const bool past = s_at < 0;
                const int sl = past ? s_last : s_at;
                const double left = past ? __builtin_inf() : want - s_base;
                __syncthreads();
                if (tid == 0) s_at = s_last = -1;
                double w[VE], s = 0, all;
                weights16<DT, PROBS>(a, S, sl * VERIFY_SLICE + tid * VE, w);
#pragma unroll
                for (int k = 0; k < VE; k++) s += w[k];
                const double e0 = block_scan(s, tmp, all);
                if (s > 0) {
                    const bool here = e0 <= left && left < e0 + s;
                    double run = e0;
                    int last = -1, at = -1;
                    for (int k = 0; k < VE; k++) {
                        if (!(w[k] > 0)) continue;
                        last = sl * VERIFY_SLICE + tid * VE + k;
                        run += w[k];
                        if (at < 0 && left < run) at = last;
                    }
                    if (here) s_at = at < 0 ? last : at;
                    atomicMax(&s_last, last);
                }
                __syncthreads();
                token = s_at < 0 ? s_last : s_at;
                break;
            }
        }
    }
    if (tid == 0) a.accepted[b] = r;
    for (int k = tid; k <= a.n; k += VT) a.tokens[b * (a.n + 1) + k] = k < r ? a.drafts[b * a.n + k] : k == r ? token : -1;
}

template <int DT, bool PROBS>
static hipError_t launch_v(const VerifyArgs & a, hipStream_t st) {
    hipLaunchKernelGGL((k_verify_rows<DT, PROBS>), dim3((unsigned) a.n_seq * (a.n + 1) * a.nsl), dim3(VT), 0, st, a);
    if (a.q && a.n) hipLaunchKernelGGL((k_verify_residual<DT, PROBS>), dim3((unsigned) a.n_seq * a.nsl), dim3(VT), 0, st, a);
    hipLaunchKernelGGL((k_verify_pick<DT, PROBS>), dim3(a.n_seq), dim3(VT), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_verify(const VerifyArgs & a, int dtype, bool probs, hipStream_t st) {
    if (probs) return launch_v<DT_F32, true>(a, st);
    return dtype == DT_F32 ? launch_v<DT_F32, false>(a, st) : dtype == DT_F16 ? launch_v<DT_F16, false>(a, st) : launch_v<DT_BF16, false>(a, st);
}

} // namespace qkv
