// How the experts' kernels (step_moe.hip) share their work: the planes' layout in LDS, parts of k for the waves, tokens and chunks of a pass.
// Host and device; the rules are the host's alone.
#pragma once
#include "step_mix_launch.h"

#include <algorithm>
#include <cmath>

namespace qkv {
namespace {

constexpr int MAX_PAIRS = MOE_ROWS * ROUTE_MAX_TOP;
constexpr int WAVES_LOG = 2, WAVES = 1 << WAVES_LOG, PER_CU = 3; // workgroups of k_moe_up and k_moe_down: their waves, and how many a CU has registers for
constexpr int OW = 16;                                           // waves of a workgroup of k_moe_down_one
constexpr int LDS_CU = 160 * 1024, ONE_LDS = 150 * 1024;         // of a CU; what k_moe_down_one takes of it at most

constexpr int planes_of(int xform) { return xform == W4_UNITS ? 1 : 3; }
constexpr int HP = 3; // of h
// operand rows of a token (three planes: the fourth stays zero), tokens in a lane's sums of an instruction, tokens of an instruction; sg: lane
// groups that share a sum are 1 << sg
constexpr int op_rows(int P) { return P == 3 ? 4 : 1; }
constexpr int lane_tokens(int P) { return 4 / op_rows(P); }
constexpr int group_of(int P, int sg) { return lane_tokens(P) << sg; }

__host__ __device__ __forceinline__ constexpr int padded(int blocks) { return (blocks + 7) & ~7; }
// a row of a plane, in memory and in LDS: [runs of 8 blocks][u][half][g][16 bytes], then 16 bytes unused: 16 rows' pieces lie in different banks
__host__ __device__ __forceinline__ constexpr int plane_bytes(int nb) { return padded(nb) * 32 + 16; }
// LDS of a pass, for `cr` runs of k at a time: token t's plane p is row t P + p; zeros for the operand's other lanes; per 32 << sg values the
// tokens' factors, and with minimums the tokens' sums
struct Lds {
    int row, zero, dx, ds, end;
};
__host__ __device__ __forceinline__ constexpr Lds lds_of(int P, int sg, int cr, int tp, bool mins) {
    Lds l{};
    l.row = cr * 256 + 16;
    l.zero = tp * P * l.row;
    l.dx = l.zero + 256;
    l.ds = l.dx + (cr * 8 >> sg) * tp * 4;
    l.end = ((mins ? l.ds + (cr * 8 >> sg) * tp * 4 : l.ds) + 15) & ~15;
    return l;
}
constexpr int WIN = 32, WROW = WIN + 8; // scales of a window, a row's place: 16 rows' 80 bytes begin in different banks
constexpr int win_bytes(int nt, bool mins) { return nt * (mins ? 2 : 1) * 16 * WROW * 2; }
inline size_t lds_bytes(const MoeArgs & a, int P, int sg, int cr, int tp) { return lds_of(P, sg, cr, tp, a.up.mins).end + (size_t) WAVES * win_bytes(2, a.up.mins); }
inline size_t one_lds(const MoeArgs & a, int P, int sg, int nt) {
    return lds_of(P, sg, padded(a.inner >> 5) >> 3, a.top_k + group_of(P, sg), a.up.mins).end + (size_t) OW * (win_bytes(nt, a.up.mins) + nt * 64);
}

// a wave's part of the runs of a chunk of k, and the chunk's first run
struct Part {
    int first, r0, r1;
};
// runs `chunk` .. of k, `cr` of them at a time, the ks-th of 1 << log parts (each has one at least: parts_hold)
__host__ __device__ __forceinline__ Part part_of(int runs, int cr, int chunk, int ks, int log) {
    const int c0 = chunk * cr, n = cr < runs - c0 ? cr : runs - c0;
    return Part{c0, c0 + ((n * ks) >> log), c0 + ((n * (ks + 1)) >> log)};
}

// lane groups that share a sum are 1 << ..: of x, and of h
inline int sg_up(const MoeArgs & a, int xform) { return planes_of(xform) == 1 ? 0 : a.gsh; }
inline int sg_down(const MoeArgs & a) { return a.ks_up == 0 ? std::min(a.gsh, 1) : 0; }
inline int runs_of(int n) { return padded(n / 32) / 8; }
// one row whose h LDS holds: its sum over the experts with the product
inline bool one_row(const MoeArgs & a) { return a.rows == 1 && one_lds(a, HP, sg_down(a), 2) <= ONE_LDS; }

// Tokens of a pass, up to 16, and runs of k that LDS holds at a time, PER_CU workgroups a CU: all of k where that leaves room for twice the tokens
// that an expert has on average, else chunks of at least four runs a wave (47 rows of 2 of 8 experts 4,096 x 8,192: 215 us, with 8 tokens
// at most 253; 3 rows of 2 of 8 of 5,120 x 6,144, two tokens with all of k 81.8, four in chunks 82.4).
inline void pass(const MoeArgs & a, int P, int sg, int runs, int ks_log, int & tp, int & cr) {
    constexpr size_t SHARE = LDS_CU / 1024 / PER_CU * 1024;
    const int tg = group_of(P, sg), least = std::min(runs, 4 << ks_log), most = std::min((std::min(a.rows, 16) + tg - 1) / tg * tg, 16);
    const int want = std::min(most, 2 * ((a.rows * a.top_k + a.n_experts - 1) / a.n_experts));
    cr = runs;
    for (tp = most; tp >= std::max(want, tg); tp -= tg)
        if (lds_bytes(a, P, sg, cr, tp) <= SHARE) return;
    for (tp = most;; tp -= tg) {
        for (cr = runs; cr > least && lds_bytes(a, P, sg, cr, tp) > SHARE;) cr = std::max(least, (cr + 1) / 2);
        if (tp <= tg || lds_bytes(a, P, sg, cr, tp) <= SHARE) break;
    }
    // (the last chunk has a run for every wave)
    while (cr < runs && runs % cr && runs % cr < 1 << ks_log) cr++;
}
// waves that split k (1 << ..): as many as leave the workgroups (of `cols` columns a wave) within one round of PER_CU a CU, as every round pays for
// its start; `experts` are those that occur
inline int split(double experts, int n, int cols, int runs, int limit) {
    int log = limit;
    while (log > 0 && (experts * ((n + (cols * WAVES >> log) - 1) / (cols * WAVES >> log)) > 256 * PER_CU || runs < 1 << log)) log--;
    return log;
}
// (of one run of at most MOE_ROWS rows)
inline void split_work(MoeArgs & a, int xform) {
    // the experts that occur where every choice is as likely as another
    const double experts = a.n_experts * (1 - std::pow(1 - 1.0 / a.n_experts, a.rows * a.top_k));
    a.ks_up = split(experts, a.inner, 16, runs_of(a.dim), WAVES_LOG - 1);
    a.ks_down = split(experts, a.dim, 32, runs_of(a.inner), WAVES_LOG);
    a.ks_one = 0;
    while (a.top_k << (a.ks_one + 1) <= OW && 1 << (a.ks_one + 1) <= runs_of(a.inner)) a.ks_one++;
    pass(a, planes_of(xform), sg_up(a, xform), runs_of(a.dim), a.ks_up, a.tp_up, a.cr_up);
    pass(a, HP, sg_down(a), runs_of(a.inner), a.ks_down, a.tp_down, a.cr_down);
}

// What the kernels take for granted of a pass: whole groups of tokens, LDS that a CU has, a run for every wave in every chunk (a wave's first loads are
// of its first and its last one), and two in all chunks but the last (both buffers of codes take the next chunk's)
inline bool parts_hold(int runs, int cr, int log) {
    if (cr < 1 || cr > runs) return false;
    for (int chunk = 0, chunks = (runs + cr - 1) / cr; chunk < chunks; chunk++)
        for (int ks = 0; ks < 1 << log; ks++) {
            const Part p = part_of(runs, cr, chunk, ks, log);
            if (p.r1 - p.r0 < (chunk + 1 < chunks ? 2 : 1) || p.r0 < 0 || p.r1 > runs) return false;
        }
    return true;
}
inline bool plan_holds(const MoeArgs & a, int xform) {
    const int P = planes_of(xform), su = sg_up(a, xform), sd = sg_down(a);
    const auto tokens = [](int tp, int tg) { return tp >= tg && tp <= 16 && tp % tg == 0; };
    if (a.ks_up < 0 || a.ks_up >= WAVES_LOG || !tokens(a.tp_up, group_of(P, su)) || !parts_hold(runs_of(a.dim), a.cr_up, a.ks_up) || lds_bytes(a, P, su, a.cr_up, a.tp_up) > LDS_CU)
        return false;
    if (one_row(a)) return a.top_k << a.ks_one <= OW && parts_hold(runs_of(a.inner), runs_of(a.inner), a.ks_one);
    return a.ks_down >= 0 && a.ks_down <= WAVES_LOG && tokens(a.tp_down, group_of(HP, sd)) && parts_hold(runs_of(a.inner), a.cr_down, a.ks_down) && lds_bytes(a, HP, sd, a.cr_down, a.tp_down) <= LDS_CU;
}

} // namespace
} // namespace qkv
