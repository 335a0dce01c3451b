// Verification of drafted tokens against the target's distribution, from given random numbers.
//
//   p_i = softmax(logits_i / T) (or the probabilities given); draft d_i is accepted while u_i q_i(d_i) < p_i(d_i), q_i the
//   draft model's probabilities, or all on d_i without one.  At the first refusal i the next token is drawn from
//   max(p_i - q_i, 0), after the last draft from p_n: the first index at which the cumulative sum of the weights exceeds
//   u_n times their total (a random number of its own: the u_i that refused a draft is not free any more).
//
// A border of the cumulative sum lies near every random number when a vocabulary's 150,000 weights are small, so weights,
// sums and the comparison are in 64 bits: the weights are within 2e-14 of themselves, two orders of summation differ by 1e-16 of
// the total, and a token changes with a probability of 1e-9.
//
// k_verify_rows: every row once, in slices of 4,096 entries (the slice's largest logit and its sum relative to that; for the
// slice of a row's draft also the sum without it).
// k_verify_residual (with q): the slices' sums of max(p - q, 0) of the one row that was refused, if any.
// k_verify_pick: one workgroup per sequence: the decision, the slice of the next token by the slices' sums, and the token
// inside the slice.
#include "step_dev.h"

namespace qkv {

constexpr int VT = 256;      // threads
constexpr int VE = VERIFY_SLICE / VT; // entries per thread

// 2^y for y <= 0 (NaN and far below: 0): y = n - f with f in [0, 1), 2^-f by its interpolation at the ten Chebyshev nodes of that
// interval, within 1.9e-14 of it (the largest difference over 2,001 points against 60 digits)
__device__ __forceinline__ double exp2_neg(double y) {
    y = __builtin_fmax(y, -2000.0);
    const double f = __builtin_amdgcn_fract(-y);
    constexpr double c[10] = {0.9999999999999901,    -0.6931471805579755,    0.24022650689399042,     -0.05550410782882977,   0.009618123647001858,
                              -0.0013333352771918547, 0.0001539881035534164, -1.5185162327257455e-05, 1.2623484285587602e-06, -7.216664926222149e-08};
    double p = c[9];
#pragma unroll
    for (int k = 8; k >= 0; k--) p = __builtin_fma(p, f, c[k]);
    return __builtin_ldexp(p, (int) y); // (towards zero)
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

// E consecutive entries of a row from j on (one load of at most 16 bytes where all of them exist); those past the end are
// `none`
template <int DT, int E> __device__ __forceinline__ void load_run(const typename Elem<DT>::T * p, int j, int vocab, float none, float (&v)[E]) {
    if (j + E <= vocab) {
        if constexpr (E == 8) load8<DT>(p + j, v);
        else Elem<DT>::load4(p + j, v);
    } else {
#pragma unroll
        for (int k = 0; k < E; k++) v[k] = j + k < vocab ? Elem<DT>::up(p[j + k]) : none;
    }
}
// entries of a thread's piece of a slice that lie together: 16 bytes of them
constexpr int run_of(int dt) { return dt == DT_F32 ? 4 : 8; }

// One row's slice: 16 entries a thread, all loads of them ahead of the first use.  What bounds it is the arithmetic in 64 bits, 26
// vector instructions an entry, 17 of them the exponential (64 sequences of up to 7 drafts over 150,001 fp32 logits, 173 MB: 43 us,
// 4.0 TB/s, the vector units busy for 83 to 86% of it, 39 to 47 by the clock the card keeps; workgroups that loop over slices with the next one's loads ahead: 54 to 86 us, by their registers); of few
// rows the launch (8 of 32,768: 4.2).
template <int DT, bool PROBS>
__global__ __launch_bounds__(VT) void k_verify_rows(VerifyArgs a) {
    __shared__ float top[VT / 64];
    __shared__ double sums[VT / 64], rests[VT / 64];
    __shared__ int args[VT / 64], bad[VT / 64];
    const int row = blockIdx.x / a.nsl, sl = blockIdx.x - row * a.nsl, b = row / (a.n + 1), i = row - b * (a.n + 1);
    if (i > count_of(a, b)) return; // (a row behind the sequence's last draft)
    const Temp t = temp_of(a, b);
    constexpr int E = run_of(DT);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, j0 = sl * VERIFY_SLICE + threadIdx.x * E;
    const auto at = [&](int k) { return j0 + k / E * (VT * E) + k % E; };
    float v[VE];
#pragma unroll
    for (int c = 0; c < VE / E; c++)
        load_run<DT, E>(static_cast<const typename Elem<DT>::T *>(a.target) + (long long) row * a.row_stride, at(c * E), a.vocab,
                        PROBS ? 0.f : -__builtin_inff(), *reinterpret_cast<float (*)[E]>(v + c * E));
    // the slice of a draft also leaves the draft's own value and, without q, its sum without the draft, what a refusal leaves over
    const int d = i < a.n ? a.drafts[b * a.n + i] : -1;
    float m = -__builtin_inff();
    bool wild = false; // a NaN (a maximum leaves it out)
#pragma unroll
    for (int k = 0; k < VE; k += 2) {
        wild |= __builtin_isunordered(v[k], v[k + 1]);
        m = fmaxf(fmaxf(m, v[k]), v[k + 1]);
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
    wild |= m == __builtin_inff();
    VerifyPart p{0.0, PROBS ? 0.f : m, 0};
    if (wild) p.top = __builtin_nanf("");
    else if (!PROBS && t.greedy) {
        int arg = 0x7fffffff;
#pragma unroll
        for (int k = VE - 1; k >= 0; k--) arg = v[k] == m && at(k) < a.vocab ? at(k) : arg;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) arg = min(arg, (int) shfl_xor_u((unsigned) arg, x));
        if (lane == 0) args[wave] = arg;
        __syncthreads();
        p.arg = args[0];
#pragma unroll
        for (int k = 1; k < VT / 64; k++) p.arg = min(p.arg, args[k]);
        p.sum = m > -__builtin_inff() ? 1.0 : 0.0;
    } else {
        const bool holds = d >= 0 && d / VERIFY_SLICE == sl && d < a.vocab;
        double s = 0;
        if (holds) { // (on its own: the selects cost every slice a quarter more)
            p.arg = __builtin_bit_cast(int, Elem<DT>::up(static_cast<const typename Elem<DT>::T *>(a.target)[(long long) row * a.row_stride + d]));
            double rest = 0;
            if (PROBS || m > -__builtin_inff()) {
#pragma unroll
                for (int k = 0; k < VE; k++) {
                    const double w = weight<PROBS>(v[k], m, t.beta);
                    s += w;
                    rest += at(k) != d ? w : 0.0;
                }
            }
            rest = wave_sum(rest);
            if (lane == 0) rests[wave] = rest;
        } else if (PROBS || m > -__builtin_inff()) {
#pragma unroll
            for (int k = 0; k < VE; k++) s += weight<PROBS>(v[k], m, t.beta);
        }
        s = wave_sum(s);
        if (lane == 0) sums[wave] = s;
        __syncthreads();
        p.sum = sums[0];
#pragma unroll
        for (int k = 1; k < VT / 64; k++) p.sum += sums[k];
        if (holds && threadIdx.x == 0) {
            double rest = rests[0];
            for (int k = 1; k < VT / 64; k++) rest += rests[k];
            if (!a.q) a.rest[row] = rest;
        }
    }
    if (threadIdx.x == 0) a.part[(size_t) row * a.nsl + sl] = p;
}

// what every workgroup of a sequence finds from the slices' sums
struct Verdict {
    float top[VERIFY_MAX_DRAFTS + 1]; // per row: the largest logit
    double z[VERIFY_MAX_DRAFTS + 1];  // the sum of the weights relative to it (probabilities: their sum); 0: not a row to draw from
    int arg[VERIFY_MAX_DRAFTS + 1];
    float p[VERIFY_MAX_DRAFTS];       // the drafts' probabilities
    int ok[VERIFY_MAX_DRAFTS];        // accepted on its own
    int draft[VERIFY_MAX_DRAFTS];     // -1: outside the vocabulary
    double less[VERIFY_MAX_DRAFTS];   // without q: the draft's slice without it, relative to the row's largest logit
};

// what a wave reads of one row: its first 64 slices, one a lane, and what belongs to its draft
struct RowIn {
    VerifyPart part;
    int d; // the draft, -1 outside the vocabulary
    float u, q;
    double rest;
};
__device__ __forceinline__ RowIn load_row(const VerifyArgs & a, int b, int i) {
    const long long row = (long long) b * (a.n + 1) + i;
    const int lane = threadIdx.x & 63;
    RowIn in{{0.0, -__builtin_inff(), 0x7fffffff}, -1, 0.f, 1.f, 0.0};
    if (lane < a.nsl) in.part = a.part[row * a.nsl + lane];
    if (i < a.n) {
        const int d = a.drafts[b * a.n + i];
        in.u = a.u[row];
        if (!a.q) in.rest = a.rest[row];
        if (d >= 0 && d < a.vocab) {
            in.d = d;
            if (a.q) in.q = a.q[((size_t) b * a.n + i) * a.vocab + d];
        }
    }
    return in;
}

// a wave per row, all NT threads; count and t: the sequence's drafts and temperature; kept (optional): [row][64] the weights
// of the rows' first 64 slices; returns the accepted count in every thread
template <bool PROBS, int NT>
__device__ __forceinline__ int decide(const VerifyArgs & a, int b, int & count, Temp & t, Verdict & V, double * kept) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const float ninf = -__builtin_inff();
    // (ahead of the sequence's own values: one wait for all of them.  A row behind the last draft is memory of the workspace
    // all the same, and what it holds is not used)
    RowIn in;
    if (wave <= a.n) in = load_row(a, b, wave);
    count = count_of(a, b);
    t = temp_of(a, b);
    for (int i = wave; i <= count; i += NT / 64) {
        if (i != wave) in = load_row(a, b, i);
        const VerifyPart * pp = a.part + ((long long) b * (a.n + 1) + i) * a.nsl;
        float m = in.part.top;
        bool wild = m != m;
        for (int s = lane + 64; s < a.nsl; s += 64) {
            const float x = pp[s].top;
            wild |= x != x;
            m = fmaxf(m, x);
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, shfl_xor(m, x));
        wild = __ballot(wild) != 0;
        double z = 0;
        int arg = 0x7fffffff;
        const auto add = [&](const VerifyPart & x) {
            if (!PROBS && t.greedy) {
                if (x.top == m) arg = min(arg, x.arg);
            } else if (x.sum > 0) z += PROBS ? x.sum : x.sum * exp2_neg(((double) x.top - (double) m) * t.beta);
        };
        add(in.part);
        if (kept) kept[i * 64 + lane] = z;
        for (int s = lane + 64; s < a.nsl; s += 64) add(pp[s]);
        if (!PROBS && t.greedy) {
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) arg = min(arg, (int) shfl_xor_u((unsigned) arg, x));
            z = m > ninf ? 1.0 : 0.0;
        } else z = wave_sum(z);
        if (wild || !(z < (double) __builtin_inff())) z = 0;
        double pd = 0, less = in.rest;
        if (i < count && in.d >= 0 && z > 0) {
            if (!PROBS && t.greedy) pd = in.d == arg ? 1.0 : 0.0;
            else {
                const int sl = __builtin_amdgcn_readfirstlane(in.d / VERIFY_SLICE);
                const int own = sl < 64 ? __builtin_amdgcn_readlane(in.part.arg, sl) : pp[sl].arg;
                pd = weight<PROBS>(__builtin_bit_cast(float, own), m, t.beta);
                if (!PROBS) {
                    pd /= z;
                    const float top = sl < 64 ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, in.part.top), sl)) : pp[sl].top;
                    less = less > 0 ? less * exp2_neg(((double) top - (double) m) * t.beta) : 0.0; // (-infinity: a slice of masked entries)
                }
            }
        }
        if (lane == 0) {
            V.top[i] = m;
            V.z[i] = z;
            V.arg[i] = arg;
            if (i < count) {
                V.draft[i] = in.d;
                V.p[i] = (float) pd;
                V.ok[i] = (double) in.u * (double) in.q < pd;
                // (below it, the slice's sum could have a weight where each entry's alone is zero)
                V.less[i] = less > 1e-290 ? less : 0.0;
            }
        }
    }
    __syncthreads();
    const uint64_t no = ~__ballot(lane < count && V.ok[lane < count ? lane : 0]);
    return min(count, no ? (int) __builtin_ctzll(no) : 64);
}

// the weights of E entries of the row the next token is drawn from
struct Source {
    long long row;   // of the target
    const float * q; // subtracted, or null
    float top;
    double beta, zinv;
    int skip;        // an entry that counts as zero (-1: none)
};
template <int DT, bool PROBS, int E>
__device__ __forceinline__ void weights(const VerifyArgs & a, const Source & S, int j, double (&w)[E]) {
    float v[E], q[E];
    load_run<DT, E>(static_cast<const typename Elem<DT>::T *>(a.target) + S.row * a.row_stride, j, a.vocab, PROBS ? 0.f : -__builtin_inff(), v);
    if (S.q) load_run<DT_F32, E>(S.q, j, a.vocab, 0.f, q);
#pragma unroll
    for (int k = 0; k < E; k++) w[k] = j + k == S.skip ? 0.0 : weight<PROBS>(v[k], S.top, S.beta);
    if (S.q) {
#pragma unroll
        for (int k = 0; k < E; k++) {
            const double r = (PROBS ? w[k] : w[k] * S.zinv) - (double) q[k];
            w[k] = r > 0 ? r : 0.0;
        }
    }
}

// (4 sequences of 3 drafts over 150,001 bf16 logits: 5.4 us, most of them the slices' sums, the decision and the refused row one
// after the other)
template <int DT, bool PROBS>
__global__ __launch_bounds__(VT) void k_verify_residual(VerifyArgs a) {
    __shared__ Verdict V;
    __shared__ double sums[VT / 64];
    const int b = blockIdx.x / a.nsl, sl = blockIdx.x - b * a.nsl;
    int count;
    Temp t;
    const int r = decide<PROBS, VT>(a, b, count, t, V, nullptr);
    if ((!PROBS && t.greedy) || r == count || !(V.z[r] > 0)) return;
    const Source S{(long long) b * (a.n + 1) + r, a.q + ((size_t) b * a.n + r) * a.vocab, V.top[r], t.beta, 1.0 / V.z[r], -1};
    constexpr int E = run_of(DT);
    double s = 0;
#pragma unroll
    for (int c = 0; c < VE / E; c++) {
        double w[E];
        weights<DT, PROBS, E>(a, S, sl * VERIFY_SLICE + (c * VT + threadIdx.x) * E, w);
#pragma unroll
        for (int k = 0; k < E; k++) s += w[k];
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = sums[0];
        for (int k = 1; k < VT / 64; k++) s += sums[k];
        a.rest[(size_t) b * a.nsl + sl] = s;
    }
}

// inclusive sum over the lanes: within rows of 16, then the rows' last values over the next row, the first half's over the second
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_d(double v) { // (0 where the lane has no source)
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const unsigned lo = (unsigned) __builtin_amdgcn_update_dpp(0, (int) (unsigned) x, CTRL, ROWS, 0xf, false),
                   hi = (unsigned) __builtin_amdgcn_update_dpp(0, (int) (unsigned) (x >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_d<0x111, 0xf>(v); // row_shr 1, 2, 4, 8
    v += dpp_d<0x112, 0xf>(v);
    v += dpp_d<0x114, 0xf>(v);
    v += dpp_d<0x118, 0xf>(v);
    v += dpp_d<0x142, 0xa>(v); // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
    v += dpp_d<0x143, 0xc>(v);
    return v;
}

// What bounds the pick is its chain: the slices' sums, the decision, one slice's entries, two scans (one sequence of 7 drafts over 32,768:
// 5.9 us, 64 over 150,001: 7.5).
constexpr int PT = 512; // threads of the pick: a wave per row, eight entries of the slice per thread (1,024: 0.4 us more, two waves more a SIMD)
constexpr int PE = VERIFY_SLICE / PT;

template <int DT, bool PROBS>
__global__ __launch_bounds__(PT) void k_verify_pick(VerifyArgs a) {
    __shared__ Verdict V;
    __shared__ double sums[PT / 64];
    __shared__ double kept[(VERIFY_MAX_DRAFTS + 1) * 64];
    __shared__ int s_at, s_last, s_slice, s_pass;
    __shared__ double s_left;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float u32 = a.u[(long long) b * (a.n + 1) + a.n];
    if (tid == 0) s_at = s_last = s_slice = -1;
    const double first = a.q && lane < a.nsl ? a.rest[(size_t) b * a.nsl + lane] : 0.0; // (of up to 64 slices)
    int count;
    Temp t;
    const int r = decide<PROBS, PT>(a, b, count, t, V, kept);
    int token = -1;
    if (V.z[r] > 0) {
        if (!PROBS && t.greedy) token = V.arg[r];
        else {
            const long long row = (long long) b * (a.n + 1) + r;
            const VerifyPart * pp = a.part + row * a.nsl;
            Source S{row, nullptr, V.top[r], t.beta, a.q ? 1.0 / V.z[r] : 1.0, -1};
            double less = 0; // the refused draft's slice without it
            if (r < count) {
                if (a.q) S.q = a.q + ((size_t) b * a.n + r) * a.vocab;
                else if ((S.skip = V.draft[r]) >= 0) less = V.less[r];
            }
            // the slice, by the first wave: lane l holds `per` slices from l per on
            const int per = (a.nsl + 63) / 64;
            Source R = S;
            for (int pass = 0; wave == 0 && pass < 2; pass++) { // (again without q and skip where they leave nothing)
                const auto slice = [&](int s) -> double {
                    if (s >= a.nsl) return 0.0;
                    if (R.q) return per == 1 ? first : a.rest[(size_t) b * a.nsl + s];
                    if (R.skip >= 0 && s == R.skip / VERIFY_SLICE) return less;
                    if (per == 1) return kept[r * 64 + s];
                    const double x = pp[s].sum;
                    return PROBS ? x : x > 0 ? x * exp2_neg(((double) pp[s].top - (double) S.top) * S.beta) : 0.0;
                };
                double mine = 0;
#pragma unroll 1
                for (int k = 0; k < per; k++) mine += slice(lane * per + k);
                const double incl = wave_scan(mine), total = __shfl(incl, 63, 64);
                if (!(total > 0)) {
                    R.q = nullptr;
                    R.skip = -1;
                    continue;
                }
                double ex = __shfl_up(incl, 1, 64); // (a lane's sum begins exactly where the one before it ends)
                if (lane == 0) ex = 0;
                const double want = (double) u32 * total;
                const uint64_t in = __ballot(mine > 0 && ex <= want && want < incl), any = __ballot(mine > 0);
                // (none, for a random number of 1 or more: the last slice with a weight, and its last entry)
                const int l = in ? (int) __builtin_ctzll(in) : 63 - (int) __builtin_clzll(any);
                int sl = lane;
                if (per > 1) {
                    sl = -1;
                    double run = ex;
#pragma unroll 1
                    for (int k = 0; k < per; k++) {
                        const double x = slice(lane * per + k);
                        if (!(x > 0)) continue;
                        if (sl >= 0 && in && want < run) break;
                        if (sl >= 0) ex = run;
                        sl = lane * per + k;
                        run += x;
                    }
                }
                if (lane == l) {
                    s_slice = sl;
                    s_pass = pass;
                    s_left = in ? want - ex : __builtin_inf();
                }
                break;
            }
            __syncthreads();
            const int sl = s_slice;
            if (sl >= 0) {
                const double left = s_left;
                if (s_pass) {
                    S.q = nullptr;
                    S.skip = -1;
                }
                double w[PE], s = 0;
                weights<DT, PROBS, PE>(a, S, sl * VERIFY_SLICE + tid * PE, w);
#pragma unroll
                for (int k = 0; k < PE; k++) s += w[k];
                const double part = wave_scan(s);
                if (lane == 63) sums[wave] = part;
                __syncthreads();
                double base = 0;
#pragma unroll
                for (int k = 0; k < PT / 64; k++) base += k < wave ? sums[k] : 0.0; // (one after the other, as every wave adds them)
                const double end = base + part;
                double begin = __shfl_up(end, 1, 64);
                if (lane == 0) begin = base;
                if (s > 0 && begin <= left && left < end) { // one thread, if any
                    double at = begin;
                    int last = -1, found = -1;
#pragma unroll
                    for (int k = 0; k < PE; k++) {
                        if (!(w[k] > 0)) continue;
                        last = sl * VERIFY_SLICE + tid * PE + k;
                        at += w[k];
                        if (found < 0 && left < at) found = last;
                    }
                    s_at = found < 0 ? last : found;
                }
                const uint64_t some = __ballot(s > 0);
                if (some && lane == 63 - (int) __builtin_clzll(some)) {
                    int last = -1;
#pragma unroll
                    for (int k = 0; k < PE; k++) last = w[k] > 0 ? sl * VERIFY_SLICE + tid * PE + k : last;
                    atomicMax(&s_last, last);
                }
                __syncthreads();
                token = s_at < 0 ? s_last : s_at;
            }
        }
    }
    if (tid == 0) a.accepted[b] = r;
    if (tid <= a.n) a.tokens[(long long) b * (a.n + 1) + tid] = tid < r ? a.drafts[b * a.n + tid] : tid == r ? token : -1;
    if (a.p && tid < a.n) a.p[(long long) b * a.n + tid] = tid < count ? V.p[tid] : 0.f;
}

template <int DT, bool PROBS>
static hipError_t launch_v(const VerifyArgs & a, hipStream_t st) {
    hipError_t e = launch(k_verify_rows<DT, PROBS>, dim3((unsigned) a.n_seq * (a.n + 1) * a.nsl), dim3(VT), 0, st, a);
    if (e == hipSuccess && a.q && a.n) e = launch(k_verify_residual<DT, PROBS>, dim3((unsigned) a.n_seq * a.nsl), dim3(VT), 0, st, a);
    if (e == hipSuccess) e = launch(k_verify_pick<DT, PROBS>, dim3(a.n_seq), dim3(PT), 0, st, a);
    return e;
}

hipError_t launch_verify(const VerifyArgs & a, int dtype, bool probs, hipStream_t st) {
    if (probs) return launch_v<DT_F32, true>(a, st);
    return dtype == DT_F32 ? launch_v<DT_F32, false>(a, st) : dtype == DT_F16 ? launch_v<DT_F16, false>(a, st) : launch_v<DT_BF16, false>(a, st);
}

} // namespace qkv
