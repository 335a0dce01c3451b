// The operators of a server of many requests beside the 4-bit products (step_lora.hip, step_route.hip, step_moe.hip): their
// arguments, checked by the C-ABI host code (step_mix_api.cpp), and their launchers.
#pragma once
#include "step_launch.h"

namespace qkv {

// y[m] = base[m] + scales[a] B_a (A_a x[m]), a = ids[m]; rows whose a is no adapter: y[m] = base[m]
struct LoraArgs {
    const void * a;      // [n_adapters][rank][k] fp16 or bf16
    const void * b;      // [n_adapters][n][rank]
    const int * ranks;   // optional [n_adapters]: the first ranks[a] of an adapter's (clamped to 0 .. rank)
    const float * scales; // optional [n_adapters]
    const int * ids;     // [rows]
    const int8_t * xa;   // int8 units [rows][k / 32][16] (a / b), meta [rows][k / 32][4]; or
    const int8_t * xb;
    const uint16_t * xmeta;
    const void * x;      // plain rows [rows][x_stride]
    const float * base;  // optional [rows][base_stride] (may be y)
    float * y;           // [rows][y_stride]
    float * u;           // workspace [chunks][rows][rp]: A x by chunks of k
    long long x_stride, base_stride, y_stride;
    int rows, n, k, n_adapters, rank;
    int rp, chunks, slots; // (set by lora_plan) rank padded to 16; chunks of k; adapters of a tile of 16 rows side by side
};
// Up to so many rows tiles of 16, whose adapters have workgroups of their own; from there tiles of 32, one workgroup for all of a tile's.  5,120 x 6,144,
// rank 16, bf16, the first and the second: 320 rows of as many requests 40 and 111 us, 1,024 87 and 156; of 8 rows a request 17 and 29, 34 and 41; of 60
// 18 and 21, 27 and 26; of one 18 and 17, 22 and 23.
constexpr int LORA_FEW_ROWS = 1024;
// Up to so many rows k is cut as if a tile's rows had an adapter each, from there as if it had LORA_TILE_ADAPTERS (512 rows of one request 22 and 19 us, of 8
// rows a request 22 and 19, of as many requests 47 and 52).
constexpr int LORA_SINGLE_ROWS = 256, LORA_TILE_ADAPTERS = 4;
constexpr int LORA_MAX_ROWS = 1 << 19, LORA_MAX_N = 1 << 24, LORA_MAX_K = 1 << 20, LORA_MAX_RANK = 256, LORA_MAX_CHUNKS = 16;
void lora_plan(LoraArgs & a);
hipError_t launch_lora(const LoraArgs & a, int xform, int wtype, hipStream_t st); // xform: W4_UNITS or a Dtype

// logits = x W^T (sums in 64 bits), the top_k experts of each row and their weights
enum { ROUTE_SOFTMAX = 0, ROUTE_CHOSEN = 1, ROUTE_SIGMOID = 2, ROUTE_SIGMOID_NORM = 3 };
struct RouteArgs {
    const void * x;     // [rows][x_stride]
    const void * w;     // [n_experts][dim]
    const float * bias; // optional [n_experts]
    float * logits;     // [rows][n_experts]
    int * ids;          // [rows][top_k]
    float * weights;    // [rows][top_k]
    double * part;      // workspace [chunks][rows][n_experts] where chunks > 1
    long long x_stride;
    int rows, dim, n_experts, top_k, form;
    float scale;
    int chunks;         // (set by route_plan) parts of dim with partial sums of their own
    int buffers;        // (set by the launcher) of values in LDS
};
constexpr int ROUTE_MAX_EXPERTS = 1024, ROUTE_MAX_TOP = 16, ROUTE_MAX_ROWS = 1 << 19, ROUTE_MAX_DIM = 1 << 17, ROUTE_MAX_CHUNKS = 8;
void route_plan(RouteArgs & a);
hipError_t launch_route(const RouteArgs & a, int dtype, int wtype, hipStream_t st);
hipError_t launch_logits(const RouteArgs & a, int dtype, int wtype, hipStream_t st); // its parts: logits, or their partial sums, ...
hipError_t launch_pick(const RouteArgs & a, hipStream_t st);                         // ... and the choice

// 4-bit weights of every expert: codes [n_experts][n][k / 2], scales and minimums [n_experts][n][gs]
struct MoeWeights {
    const uint8_t * codes;
    const uint16_t * scales;
    const uint16_t * mins;
};
struct MoeArgs {
    MoeWeights up;   // n = 2 inner (the gate's rows, then the up projection's), k = dim
    MoeWeights down; // n = dim, k = inner
    const int8_t * xa; // int8 units, or
    const int8_t * xb;
    const uint16_t * xmeta;
    const void * x;  // plain rows [rows][x_stride]
    const int * ids; // [rows][top_k]
    const float * weights;
    void * y;        // [rows][y_stride] of x's type (units: fp32)
    long long x_stride, y_stride;
    int rows, dim, inner, n_experts, top_k, gsh; // a scale serves 32 << gsh values
    // workspace (set by moe_plan).  x and h as int8 planes: of every row (h: of every pair of a row and a place among its experts) the
    // planes' rows, as LDS holds them, a factor for every exponent, and a sum
    uint8_t * lists; // the experts that occur and their pairs (step_moe.hip)
    uint8_t * xq, * hq;
    float * xd, * hd, * xs, * hs;
    float * out;     // [pairs][dim]: the experts' outputs (where xq, xd and xs were)
    // (set by the launcher) tokens of an expert that a pass holds in LDS, runs of k that it holds at a time, and waves (1 << ..) that split k
    int tp_up, tp_down, cr_up, cr_down, ks_up, ks_down, ks_one;
};
constexpr int MOE_ROWS = 64, MOE_PICK = 256; // rows of a run; a call of more runs them one after another; experts that it can choose from itself
constexpr int MOE_MAX_ROWS = 4096, MOE_MAX_DIM = 16384, MOE_MAX_INNER = 32768;
long long moe_plan(MoeArgs & a, int xform, uint8_t * ws); // -> bytes of workspace
// route: the router whose logits, or their partial sums, are there and whose choice is ids and weights (null: these are given); at most MOE_ROWS
// rows and MOE_PICK experts
hipError_t launch_moe(const MoeArgs & a, int xform, const RouteArgs * route, hipStream_t st);

} // namespace qkv
