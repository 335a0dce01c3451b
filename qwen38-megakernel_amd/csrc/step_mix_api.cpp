// C ABI of the adapters of many requests, the router and the mixture of experts: the checks of their arguments and their launches.  They
// hold no state and no memory of their own; errors as in kv_api.cpp.
#include "../../include/qwen38_kv.h"
#include "step_check.h"
#include "step_mix_launch.h"

#include <algorithm>
#include <cmath>

using namespace qkv;

namespace {

// x as int8 units or as plain rows
template <class A> void check_x(const A & a, int xform) {
    if (xform == W4_UNITS) {
        need(a.xa, "q32a");
        need(a.xb, "q32b");
        need(a.xmeta, "q32meta");
        aligned(a.xa, 16, "q32a");
        aligned(a.xb, 16, "q32b");
        aligned(a.xmeta, 8, "q32meta");
    } else {
        need(a.x, "x");
        aligned(a.x, size_of(xform), "x");
    }
}
template <class A> void hold_x(const Device & d, const A & a) {
    d.holds(a.xa, "x (a)");
    d.holds(a.xb, "x (b)");
    d.holds(a.xmeta, "x (meta)");
    d.holds(a.x, "x");
}
void check_ws(const void * ws, long long ws_bytes, long long want, const char * of) {
    if (!ws || ws_bytes < want) bad("the call needs " + std::to_string(want) + " bytes of workspace (" + of + ")");
    aligned(ws, 16, "ws");
}

// The most bytes that calls of lo .. hi rows need, where plan(rows) gives a call of `max` parts at most and never more of more rows: of each number
// of parts the most rows that still have it.
template <class Plan, class Bytes> long long most_bytes(int lo, int hi, int max, Plan plan, Bytes bytes) {
    long long most = 0;
    for (int parts = 1; parts <= max && lo <= hi; parts++) {
        if (plan(lo).chunks < parts) break;
        int at = lo, end = hi; // plan(at) has as many
        while (at < end) {
            const int mid = at + (end - at + 1) / 2;
            if (plan(mid).chunks >= parts) at = mid;
            else end = mid - 1;
        }
        most = std::max(most, bytes(plan(at)));
    }
    return most;
}

// ------------------------------------------------------------------------------------------------ adapters
void lora_shape(int rows, int k, int rank) {
    if (rows < 0 || rows > LORA_MAX_ROWS) bad("rows outside 0 .. 524288");
    if (k < 32 || k > LORA_MAX_K || k % 32) bad("k must be a multiple of 32, at most 2^20");
    if (rank < 1 || rank > LORA_MAX_RANK) bad("rank outside 1 .. 256");
}
long long lora_ws(const LoraArgs & a) { return (long long) a.chunks * a.rows * a.rp * 4; }
// of up to `rows` rows: a workspace serves every smaller call too
long long lora_ws_upto(int rows, int k, int rank) {
    const auto plan = [&](int r) {
        LoraArgs a{};
        a.rows = r;
        a.k = k;
        a.rank = rank;
        lora_plan(a);
        return a;
    };
    return std::max({most_bytes(1, std::min(rows, LORA_SINGLE_ROWS), LORA_MAX_CHUNKS, plan, lora_ws),
                     most_bytes(LORA_SINGLE_ROWS + 1, std::min(rows, LORA_FEW_ROWS), LORA_MAX_CHUNKS, plan, lora_ws),
                     most_bytes(LORA_FEW_ROWS + 1, rows, LORA_MAX_CHUNKS, plan, lora_ws)});
}

int lora(LoraArgs a, int ab_dtype, int xform, void * ws, long long ws_bytes, void * stream) {
    lora_shape(a.rows, a.k, a.rank);
    if (xform == W4_UNITS && a.k % 64) bad("k must be a multiple of 64, at most 2^20");
    if (a.n < 1 || a.n > LORA_MAX_N) bad("n outside 1 .. 2^24");
    if (a.n_adapters < 1) bad("n_adapters is less than 1");
    if (ab_dtype != DT_F16 && ab_dtype != DT_BF16) bad("ab_dtype: 1 fp16, 2 bf16");
    if ((long long) a.rows * a.n > 1ll << 35) bad("too many results in one call");
    if (a.y_stride < a.n) bad("y_stride is less than n");
    if (a.base && a.base_stride < a.n) bad("base_stride is less than n");
    if (a.base && a.base == a.y && a.base_stride != a.y_stride) bad("y in place of base needs its stride");
    if (!a.rows) return 0; // (an empty tensor's pointers are null)
    check_x(a, xform);
    need(a.a, "a");
    need(a.b, "b");
    need(a.ids, "ids");
    need(a.y, "y");
    aligned(a.a, 2, "a");
    aligned(a.b, 2, "b");
    for (const void * p : {(const void *) a.ranks, (const void *) a.scales, (const void *) a.ids, (const void *) a.base, (const void *) a.y})
        aligned(p, 4, "an array of 4-byte values");
    lora_plan(a);
    check_ws(ws, ws_bytes, lora_ws(a), "mk_lora_ws");
    a.u = static_cast<float *>(ws);
    const Device d(stream);
    d.holds(a.a, "a");
    d.holds(a.b, "b");
    d.holds(a.ranks, "ranks");
    d.holds(a.scales, "scales");
    d.holds(a.ids, "ids");
    hold_x(d, a);
    d.holds(a.base, "base");
    d.holds(a.y, "y");
    d.holds(ws, "ws");
    ck(launch_lora(a, xform, ab_dtype, static_cast<hipStream_t>(stream)), "lora");
    return 0;
}

LoraArgs lora_args(int rows, int n, int k, int n_adapters, int rank, const void * a, const void * b, const int * ranks, const float * scales, const int * ids,
                   const float * base, long long base_stride, float * y, long long y_stride) {
    LoraArgs l{};
    l.rows = rows;
    l.n = n;
    l.k = k;
    l.n_adapters = n_adapters;
    l.rank = rank;
    l.a = a;
    l.b = b;
    l.ranks = ranks;
    l.scales = scales;
    l.ids = ids;
    l.base = base;
    l.base_stride = base_stride;
    l.y = y;
    l.y_stride = y_stride;
    return l;
}

// ------------------------------------------------------------------------------------------------ router
void route_shape(int rows, int dim, int n_experts) {
    if (rows < 0 || rows > ROUTE_MAX_ROWS) bad("rows outside 0 .. 524288");
    if (dim < 1 || dim > ROUTE_MAX_DIM) bad("dim outside 1 .. 2^17");
    if (n_experts < 1 || n_experts > ROUTE_MAX_EXPERTS) bad("n_experts outside 1 .. 1024");
}
void top_shape(int n_experts, int top_k) {
    if (top_k < 1 || top_k > ROUTE_MAX_TOP || top_k > n_experts) bad("top_k outside 1 .. 16 or above n_experts");
}
long long route_ws(const RouteArgs & a) { return a.chunks > 1 ? (long long) a.chunks * a.rows * a.n_experts * 8 : 0; }
long long route_ws_upto(int rows, int dim, int n_experts) {
    return most_bytes(1, rows, ROUTE_MAX_CHUNKS, [&](int r) {
        RouteArgs a{};
        a.rows = r;
        a.dim = dim;
        a.n_experts = n_experts;
        route_plan(a);
        return a;
    }, route_ws);
}

void check_route(const RouteArgs & a, int dtype, int w_dtype) {
    (void) size_of(dtype);
    (void) size_of(w_dtype);
    route_shape(a.rows, a.dim, a.n_experts);
    top_shape(a.n_experts, a.top_k);
    if (a.form < ROUTE_SOFTMAX || a.form > ROUTE_SIGMOID_NORM) bad("form: 0 softmax, 1 softmax of the chosen, 2 sigmoid, 3 sigmoid over the chosen ones' sum");
    if (a.bias && a.form < ROUTE_SIGMOID) bad("a bias is for the sigmoid forms");
    if (!std::isfinite(a.scale)) bad("scale must be finite");
    if (a.x_stride < a.dim) bad("x_stride is less than dim");
}
void check_route_pointers(const RouteArgs & a, int dtype, int w_dtype) {
    need(a.x, "x");
    need(a.w, "w");
    need(a.logits, "logits");
    need(a.ids, "ids");
    need(a.weights, "weights");
    aligned(a.x, size_of(dtype), "x");
    aligned(a.w, size_of(w_dtype), "w");
    for (const void * p : {(const void *) a.bias, (const void *) a.logits, (const void *) a.ids, (const void *) a.weights}) aligned(p, 4, "an array of 4-byte values");
}
void hold_route(const Device & d, const RouteArgs & a) {
    d.holds(a.x, "x");
    d.holds(a.w, "w");
    d.holds(a.bias, "bias");
    d.holds(a.logits, "logits");
    d.holds(a.ids, "ids");
    d.holds(a.weights, "weights");
}

// ------------------------------------------------------------------------------------------------ experts
void moe_shape(int rows, int dim, int inner, int n_experts, int top_k) {
    if (rows < 0 || rows > MOE_MAX_ROWS) bad("rows outside 0 .. 4096");
    if (dim < 32 || dim > MOE_MAX_DIM || dim % 32) bad("dim must be a multiple of 32, at most 16384");
    if (inner < 32 || inner > MOE_MAX_INNER || inner % 32) bad("inner must be a multiple of 32, at most 32768");
    if (n_experts < 1 || n_experts > ROUTE_MAX_EXPERTS) bad("n_experts outside 1 .. 1024");
    top_shape(n_experts, top_k);
}
long long up256(long long n) { return (n + 255) & ~255ll; }

MoeArgs moe_args(int rows, int dim, int inner, int n_experts, int top_k, int group, const void * up, const void * up_scales, const void * up_mins,
                 const void * down, const void * down_scales, const void * down_mins, const int * ids, const float * weights, void * y, long long y_stride) {
    MoeArgs a{};
    a.rows = rows;
    a.dim = dim;
    a.inner = inner;
    a.n_experts = n_experts;
    a.top_k = top_k;
    a.gsh = group == 32 ? 0 : group == 64 ? 1 : group == 128 ? 2 : -1;
    a.up = {static_cast<const uint8_t *>(up), static_cast<const uint16_t *>(up_scales), static_cast<const uint16_t *>(up_mins)};
    a.down = {static_cast<const uint8_t *>(down), static_cast<const uint16_t *>(down_scales), static_cast<const uint16_t *>(down_mins)};
    a.ids = ids;
    a.weights = weights;
    a.y = y;
    a.y_stride = y_stride;
    return a;
}
void check_moe(const MoeArgs & a, int xform) {
    moe_shape(a.rows, a.dim, a.inner, a.n_experts, a.top_k);
    if (a.gsh < 0) bad("group must be 32, 64 or 128");
    if (xform == W4_UNITS) {
        if (a.dim % 64) bad("units need a dim that is a multiple of 64");
    } else {
        (void) size_of(xform);
        if (a.x_stride < a.dim) bad("x_stride is less than dim");
    }
    if (a.y_stride < a.dim) bad("y_stride is less than dim");
    if ((a.up.mins != nullptr) != (a.down.mins != nullptr)) bad("minimums of both products or of none");
}
void check_moe_pointers(const MoeArgs & a, int xform) {
    check_x(a, xform);
    need(a.up.codes, "up");
    need(a.up.scales, "up_scales");
    need(a.down.codes, "down");
    need(a.down.scales, "down_scales");
    need(a.ids, "ids");
    need(a.weights, "weights");
    need(a.y, "y");
    aligned(a.up.codes, 16, "up");
    aligned(a.down.codes, 16, "down");
    for (const void * p : {(const void *) a.up.scales, (const void *) a.up.mins, (const void *) a.down.scales, (const void *) a.down.mins}) aligned(p, 2, "a scale array");
    aligned(a.ids, 4, "ids");
    aligned(a.weights, 4, "weights");
    aligned(a.y, xform == W4_UNITS ? 4 : size_of(xform), "y");
}
void hold_moe(const Device & d, const MoeArgs & a) {
    hold_x(d, a);
    d.holds(a.up.codes, "up");
    d.holds(a.up.scales, "up_scales");
    d.holds(a.up.mins, "up_mins");
    d.holds(a.down.codes, "down");
    d.holds(a.down.scales, "down_scales");
    d.holds(a.down.mins, "down_mins");
    d.holds(a.ids, "ids");
    d.holds(a.weights, "weights");
    d.holds(a.y, "y");
}
int moe(MoeArgs a, int xform, void * ws, long long ws_bytes, void * stream) {
    check_moe(a, xform);
    if (!a.rows) return 0; // (an empty tensor's pointers are null)
    check_moe_pointers(a, xform);
    check_ws(ws, ws_bytes, moe_plan(a, xform, static_cast<uint8_t *>(ws)), "mk_moe_ws");
    const Device d(stream);
    hold_moe(d, a);
    d.holds(ws, "ws");
    ck(launch_moe(a, xform, nullptr, static_cast<hipStream_t>(stream)), "moe");
    return 0;
}

} // namespace

extern "C" {

long long mk_lora_ws(int rows, int k, int rank) {
    return guarded<long long>([&] {
        lora_shape(rows, k, rank);
        return lora_ws_upto(rows, k, rank);
    });
}

int mk_lora_rows(int rows, int n, int k, int n_adapters, int rank, const void * a, const void * b, int ab_dtype, const int * ranks, const float * scales,
                 const int * ids, const void * x, long long x_stride, int dtype, const float * base, long long base_stride, float * y, long long y_stride,
                 void * ws, long long ws_bytes, void * stream) {
    return guarded<int>([&] {
        (void) size_of(dtype);
        if (x_stride < k) bad("x_stride is less than k");
        LoraArgs l = lora_args(rows, n, k, n_adapters, rank, a, b, ranks, scales, ids, base, base_stride, y, y_stride);
        l.x = x;
        l.x_stride = x_stride;
        return lora(l, ab_dtype, dtype, ws, ws_bytes, stream);
    });
}

int mk_lora_units(int rows, int n, int k, int n_adapters, int rank, const void * a, const void * b, int ab_dtype, const int * ranks, const float * scales,
                  const int * ids, const void * q32a, const void * q32b, const unsigned short * q32meta, const float * base, long long base_stride, float * y,
                  long long y_stride, void * ws, long long ws_bytes, void * stream) {
    return guarded<int>([&] {
        LoraArgs l = lora_args(rows, n, k, n_adapters, rank, a, b, ranks, scales, ids, base, base_stride, y, y_stride);
        l.xa = static_cast<const int8_t *>(q32a);
        l.xb = static_cast<const int8_t *>(q32b);
        l.xmeta = q32meta;
        return lora(l, ab_dtype, W4_UNITS, ws, ws_bytes, stream);
    });
}

long long mk_moe_route_ws(int rows, int dim, int n_experts) {
    return guarded<long long>([&] {
        route_shape(rows, dim, n_experts);
        return route_ws_upto(rows, dim, n_experts);
    });
}

int mk_moe_route(int rows, int dim, int n_experts, int top_k, const void * x, long long x_stride, int dtype, const void * w, int w_dtype, const float * bias,
                 int form, float scale, float * logits, int * ids, float * weights, void * ws, long long ws_bytes, void * stream) {
    return guarded<int>([&] {
        RouteArgs a{x, w, bias, logits, ids, weights, nullptr, x_stride, rows, dim, n_experts, top_k, form, scale, 1};
        check_route(a, dtype, w_dtype);
        if (!rows) return 0; // (an empty tensor's pointers are null)
        check_route_pointers(a, dtype, w_dtype);
        route_plan(a);
        const long long want = route_ws(a);
        if (want) check_ws(ws, ws_bytes, want, "mk_moe_route_ws");
        a.part = static_cast<double *>(ws);
        const Device d(stream);
        hold_route(d, a);
        if (want) d.holds(ws, "ws");
        ck(launch_route(a, dtype, w_dtype, static_cast<hipStream_t>(stream)), "route");
        return 0;
    });
}

long long mk_moe_ws(int rows, int dim, int inner, int n_experts, int top_k) {
    return guarded<long long>([&] {
        moe_shape(rows, dim, inner, n_experts, top_k);
        MoeArgs a{};
        a.rows = rows;
        a.dim = dim;
        a.inner = inner;
        a.n_experts = n_experts;
        a.top_k = top_k;
        a.up.mins = reinterpret_cast<const uint16_t *>(8); // (the form that needs most)
        return up256(route_ws_upto(rows, dim, n_experts)) + moe_plan(a, DT_F32, nullptr); // (which never falls with the rows)
    });
}

int mk_moe_rows(int rows, int dim, int inner, int n_experts, int top_k, int group, const void * up, const void * up_scales, const void * up_mins,
                const void * down, const void * down_scales, const void * down_mins, const void * x, long long x_stride, int dtype, const int * ids,
                const float * weights, void * y, long long y_stride, void * ws, long long ws_bytes, void * stream) {
    return guarded<int>([&] {
        MoeArgs a = moe_args(rows, dim, inner, n_experts, top_k, group, up, up_scales, up_mins, down, down_scales, down_mins, ids, weights, y, y_stride);
        a.x = x;
        a.x_stride = x_stride;
        (void) size_of(dtype);
        return moe(a, dtype, ws, ws_bytes, stream);
    });
}

int mk_moe_units(int rows, int dim, int inner, int n_experts, int top_k, int group, const void * up, const void * up_scales, const void * up_mins,
                 const void * down, const void * down_scales, const void * down_mins, const void * q32a, const void * q32b, const unsigned short * q32meta,
                 const int * ids, const float * weights, float * y, long long y_stride, void * ws, long long ws_bytes, void * stream) {
    return guarded<int>([&] {
        MoeArgs a = moe_args(rows, dim, inner, n_experts, top_k, group, up, up_scales, up_mins, down, down_scales, down_mins, ids, weights, y, y_stride);
        a.xa = static_cast<const int8_t *>(q32a);
        a.xb = static_cast<const int8_t *>(q32b);
        a.xmeta = q32meta;
        return moe(a, W4_UNITS, ws, ws_bytes, stream);
    });
}

int mk_moe_layer(int rows, int dim, int inner, int n_experts, int top_k, int group, const void * up, const void * up_scales, const void * up_mins,
                 const void * down, const void * down_scales, const void * down_mins, const void * x, long long x_stride, int dtype, const void * router,
                 int router_dtype, const float * bias, int form, float scale, float * logits, int * ids, float * weights, void * y, long long y_stride, void * ws,
                 long long ws_bytes, void * stream) {
    return guarded<int>([&] {
        MoeArgs a = moe_args(rows, dim, inner, n_experts, top_k, group, up, up_scales, up_mins, down, down_scales, down_mins, ids, weights, y, y_stride);
        a.x = x;
        a.x_stride = x_stride;
        RouteArgs r{x, router, bias, logits, ids, weights, nullptr, x_stride, rows, dim, n_experts, top_k, form, scale, 1};
        (void) size_of(dtype);
        check_moe(a, dtype);
        check_route(r, dtype, router_dtype);
        if (!rows) return 0; // (an empty tensor's pointers are null)
        check_route_pointers(r, dtype, router_dtype);
        check_moe_pointers(a, dtype);
        route_plan(r);
        const long long first = up256(route_ws(r));
        check_ws(ws, ws_bytes, first + moe_plan(a, dtype, static_cast<uint8_t *>(ws) + first), "mk_moe_ws");
        r.part = static_cast<double *>(ws);
        const Device d(stream);
        hold_route(d, r);
        hold_moe(d, a);
        d.holds(ws, "ws");
        // (of a few rows the choice is made where x is made ready)
        const bool few = rows <= MOE_ROWS && n_experts <= MOE_PICK;
        ck(few ? launch_logits(r, dtype, router_dtype, static_cast<hipStream_t>(stream)) : launch_route(r, dtype, router_dtype, static_cast<hipStream_t>(stream)), "route");
        ck(launch_moe(a, dtype, few ? &r : nullptr, static_cast<hipStream_t>(stream)), "moe");
        return 0;
    });
}

} // extern "C"
