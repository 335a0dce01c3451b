// The operators of a decode step around the KV store (step_norm.hip, step_w4.hip, step_verify.hip): their arguments,
// checked by the C-ABI host code (step_api.cpp), and their launchers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qkv {

enum Dtype { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };

// h = x + res; y = h / sqrt(mean(h^2) + eps) * w, as rows and / or as int8 units
struct NormArgs {
    const void * x;   // [rows][x_stride]
    const void * res; // optional [rows][res_stride]
    void * sum;       // optional [rows][sum_stride]: h (may be res)
    void * y;         // optional [rows][y_stride]
    const float * w;  // [dim]
    int8_t * a;       // optional units [rows][dim / 32][16] of the even and the odd blocks, meta [rows][dim / 32][4]
    int8_t * b;
    uint16_t * meta;
    long long x_stride, res_stride, sum_stride, y_stride;
    int rows, dim;
    float eps;
};
constexpr int NORM_MAX_DIM = 32768, NORM_MAX_ROWS = 1 << 21; // (up to 1,024 threads a row, fewer than 2^32 in a launch)
hipError_t launch_norm(const NormArgs & a, int dtype, hipStream_t st);

// y[m][j] = sum_k W[j][k] x[m][k], W[j][k] = scales[j][k >> (5 + gsh)] (code - 8) + mins[..]
struct W4Args {
    const uint8_t * codes;   // [n][k / 2]: 4-bit codes in the packed rows' word order (kv_codes.h)
    const uint16_t * scales; // [n][gs] fp16
    const uint16_t * mins;   // optional [n][gs] fp16
    const int8_t * xa;       // int8 units [rows][k / 32][16] (a / b), meta [rows][k / 32][4]; or
    const int8_t * xb;
    const uint16_t * xmeta;
    const void * x;          // plain rows [rows][x_stride]
    float * y;               // [rows][y_stride]
    long long x_stride, y_stride;
    int rows, n, k;
    int gsh, gs;             // a scale serves 32 << gsh values; gs = ceil(k / that) scales per row
    int wk_log;              // (set by the launcher) waves of a workgroup that share a tile: 1 << wk_log
    int kcb;                 // (set by the launcher) 32-value blocks of x held in LDS at a time; more than 8 rows: tiles of a workgroup
};
enum { W4_UNITS = 3 };       // launch_w4: x as int8 units, else a Dtype
hipError_t launch_w4(const W4Args & a, int xform, hipStream_t st);

// one slice of VERIFY_SLICE entries of one row of the target
struct VerifyPart {
    double sum; // of the weights, relative to the slice's largest logit (probabilities: as they are)
    float top;  // the largest logit (probabilities: 0); NaN: the slice holds a NaN or a +infinity
    int arg;    // temperature 0: the largest logit's index, the lowest of equal ones; else, in a draft's slice, the bits of its value
};
struct VerifyArgs {
    const void * target;  // [n_seq][n + 1][row_stride]
    const float * temp;   // optional [n_seq] (null: 1); 0: greedy
    const float * q;      // optional [n_seq][n][vocab]
    const int * drafts;   // [n_seq][n]
    const int * n_drafts; // optional [n_seq]
    const float * u;      // [n_seq][n + 1]
    int * accepted;       // [n_seq]
    int * tokens;         // [n_seq][n + 1]
    float * p;            // optional [n_seq][n]
    VerifyPart * part;    // [n_seq (n + 1)][nsl]
    // with q: [n_seq][nsl] sums of max(p - q, 0) of the refused row; without: [n_seq (n + 1)] per row the sum of its draft's
    // slice without the draft
    double * rest;
    long long row_stride;
    int n_seq, n, vocab, nsl;
};
constexpr int VERIFY_SLICE = 4096, VERIFY_MAX_DRAFTS = 64, VERIFY_MAX_VOCAB = 1 << 24, VERIFY_MAX_SLICES = 1 << 23;
hipError_t launch_verify(const VerifyArgs & a, int dtype, bool probs, hipStream_t st);

} // namespace qkv
