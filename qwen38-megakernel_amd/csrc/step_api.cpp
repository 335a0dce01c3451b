// C ABI of the operators of a decode step around the KV store: the checks of their arguments and their launches.  They hold
// no state and no memory of their own; errors as in kv_api.cpp.
#include "../../include/qwen38_kv.h"
#include "step_launch.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

namespace qkv {
void set_error(const char * msg); // kv_api.cpp: mk_last_error's message
}

using namespace qkv;

namespace {

template <class R, class F> R guarded(F f) {
    try {
        return f();
    } catch (const std::exception & e) {
        set_error(e.what());
    } catch (...) {
        set_error("unknown exception");
    }
    return -1;
}

[[noreturn]] void bad(const std::string & msg) { throw std::runtime_error(msg); }

void ck(hipError_t e, const char * what) {
    if (e == hipSuccess) return;
    (void) hipGetLastError(); // (reported here, not by a later call)
    bad(std::string(what) + ": " + hipGetErrorString(e));
}

// the stream is of the current device, and every buffer is memory of it (a host address or another device's would fault the GPU)
struct Device {
    int dev = -1;
    explicit Device(void * stream) {
        ck(hipGetDevice(&dev), "hipGetDevice");
        if (!stream || stream == hipStreamLegacy || stream == hipStreamPerThread) return; // (of the current device)
        hipDevice_t of = -1;
        ck(hipStreamGetDevice(static_cast<hipStream_t>(stream), &of), "stream");
        if (of != dev) bad("stream is of device " + std::to_string(of) + ", the current device is " + std::to_string(dev));
    }
    void holds(const void * p, const char * name) const {
        if (!p) return;
        hipPointerAttribute_t at{};
        const hipError_t e = hipPointerGetAttributes(&at, p);
        if (e != hipSuccess) (void) hipGetLastError(); // (reported here, not by a later call)
        if (e != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)) bad(std::string(name) + " is not device memory");
        if (at.device != dev)
            bad(std::string(name) + " is memory of device " + std::to_string(at.device) + ", the current device is " + std::to_string(dev));
    }
};

void need(const void * p, const char * name) {
    if (!p) bad(std::string("null ") + name + " pointer");
}
void aligned(const void * p, unsigned to, const char * name) {
    if ((uintptr_t) p % to) bad(std::string(name) + " is not aligned to " + std::to_string(to) + " bytes");
}
unsigned size_of(int dtype) {
    if (dtype < DT_F32 || dtype > DT_BF16) bad("dtype: 0 fp32, 1 fp16, 2 bf16");
    return dtype == DT_F32 ? 4 : 2;
}

constexpr int W4_MAX_ROWS = 1 << 19, W4_MAX_N = 1 << 28, W4_MAX_K = 1 << 20;

int w4(W4Args a, int group, int xform, void * stream) {
    if (a.rows < 0 || a.rows > W4_MAX_ROWS) bad("rows outside 0 .. 524288");
    if (a.n < 1 || a.n > W4_MAX_N) bad("n outside 1 .. 2^28");
    const int unit = xform == W4_UNITS ? 64 : 32;
    if (a.k < unit || a.k > W4_MAX_K || a.k % unit) bad("k must be a multiple of " + std::to_string(unit) + ", at most 2^20");
    if (group != 32 && group != 64 && group != 128) bad("group must be 32, 64 or 128");
    if (a.y_stride < a.n) bad("y_stride is less than n");
    a.gsh = group == 32 ? 0 : group == 64 ? 1 : 2;
    a.gs = (a.k + group - 1) / group;
    if (!a.rows) return 0; // (an empty tensor's pointers are null)
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
    need(a.codes, "codes");
    need(a.scales, "scales");
    need(a.y, "y");
    aligned(a.codes, 16, "codes");
    aligned(a.scales, 2, "scales");
    aligned(a.mins, 2, "mins");
    aligned(a.y, 4, "y");
    const Device d(stream);
    d.holds(a.codes, "codes");
    d.holds(a.scales, "scales");
    d.holds(a.mins, "mins");
    d.holds(a.xa, "x (a)");
    d.holds(a.xb, "x (b)");
    d.holds(a.xmeta, "x (meta)");
    d.holds(a.x, "x");
    d.holds(a.y, "y");
    ck(launch_w4(a, xform, static_cast<hipStream_t>(stream)), "w4");
    return 0;
}

int slices(int vocab) { return (vocab + VERIFY_SLICE - 1) / VERIFY_SLICE; }
void verify_shape(int n_seq, int n_draft, int vocab) {
    if (n_seq < 0 || n_seq > 65535) bad("n_seq outside 0 .. 65535");
    if (n_draft < 0 || n_draft > VERIFY_MAX_DRAFTS) bad("n_draft outside 0 .. 64");
    if (vocab < 1 || vocab > VERIFY_MAX_VOCAB) bad("vocab outside 1 .. 2^24");
    // (a workgroup of 256 threads per slice, fewer than 2^32 threads in a launch)
    if ((long long) n_seq * (n_draft + 1) * slices(vocab) > VERIFY_MAX_SLICES) bad("too many rows of this vocabulary in one call");
}
long long verify_ws(int n_seq, int n_draft, int vocab) {
    verify_shape(n_seq, n_draft, vocab);
    const long long nsl = slices(vocab);
    return n_seq * (nsl * (n_draft + 1) * (long long) sizeof(VerifyPart) + std::max<long long>(nsl, n_draft + 1) * (long long) sizeof(double));
}

} // namespace

extern "C" {

int mk_norm_q32(const void * x, long long x_stride, const void * res, long long res_stride, const float * w, int rows, int dim, float eps, int dtype,
                void * sum, long long sum_stride, void * y, long long y_stride, void * q32a, void * q32b, unsigned short * q32meta, void * stream) {
    return guarded<int>([&] {
        const unsigned sz = size_of(dtype);
        if (rows < 0 || rows > NORM_MAX_ROWS) bad("rows outside 0 .. 2^21");
        if (dim < 1 || dim > NORM_MAX_DIM) bad("dim outside 1 .. 32768");
        if (!(eps >= 0.f) || std::isinf(eps)) bad("eps must be finite and not negative");
        if (!rows) return 0; // (an empty tensor's pointers are null)
        if ((q32a != nullptr) != (q32b != nullptr) || (q32a != nullptr) != (q32meta != nullptr)) bad("the q32 outputs come as a set: a, b and meta");
        if (q32a && dim % 64) bad("q32 units need a dim that is a multiple of 64");
        if (!sum && !y && !q32a) bad("no output given");
        need(x, "x");
        need(w, "w");
        if (x_stride < dim) bad("x_stride is less than dim");
        if (res && res_stride < dim) bad("res_stride is less than dim");
        if (sum && sum_stride < dim) bad("sum_stride is less than dim");
        if (y && y_stride < dim) bad("y_stride is less than dim");
        if (sum && sum == res && sum_stride != res_stride) bad("sum in place of res needs its stride");
        if (y && y == x && y_stride != x_stride) bad("y in place of x needs its stride");
        aligned(x, sz, "x");
        aligned(res, sz, "res");
        aligned(sum, sz, "sum");
        aligned(y, sz, "y");
        aligned(w, 4, "w");
        aligned(q32a, 16, "q32a");
        aligned(q32b, 16, "q32b");
        aligned(q32meta, 8, "q32meta");
        const Device d(stream);
        d.holds(x, "x");
        d.holds(res, "res");
        d.holds(w, "w");
        d.holds(sum, "sum");
        d.holds(y, "y");
        d.holds(q32a, "q32a");
        d.holds(q32b, "q32b");
        d.holds(q32meta, "q32meta");
        const NormArgs a{x, res, sum, y, w, static_cast<int8_t *>(q32a), static_cast<int8_t *>(q32b), q32meta, x_stride, res_stride, sum_stride, y_stride,
                         rows, dim, eps};
        ck(launch_norm(a, dtype, static_cast<hipStream_t>(stream)), "norm");
        return 0;
    });
}

int mk_w4_units(int rows, int n, int k, int group, const void * codes, const void * scales, const void * mins, const void * q32a, const void * q32b,
                const unsigned short * q32meta, float * y, long long y_stride, void * stream) {
    return guarded<int>([&] {
        W4Args a{};
        a.codes = static_cast<const uint8_t *>(codes);
        a.scales = static_cast<const uint16_t *>(scales);
        a.mins = static_cast<const uint16_t *>(mins);
        a.xa = static_cast<const int8_t *>(q32a);
        a.xb = static_cast<const int8_t *>(q32b);
        a.xmeta = q32meta;
        a.y = y;
        a.y_stride = y_stride;
        a.rows = rows;
        a.n = n;
        a.k = k;
        return w4(a, group, W4_UNITS, stream);
    });
}

int mk_w4_rows(int rows, int n, int k, int group, const void * codes, const void * scales, const void * mins, const void * x, long long x_stride,
               int dtype, float * y, long long y_stride, void * stream) {
    return guarded<int>([&] {
        (void) size_of(dtype);
        if (x_stride < k) bad("x_stride is less than k");
        W4Args a{};
        a.codes = static_cast<const uint8_t *>(codes);
        a.scales = static_cast<const uint16_t *>(scales);
        a.mins = static_cast<const uint16_t *>(mins);
        a.x = x;
        a.x_stride = x_stride;
        a.y = y;
        a.y_stride = y_stride;
        a.rows = rows;
        a.n = n;
        a.k = k;
        return w4(a, group, dtype, stream);
    });
}

long long mk_verify_ws(int n_seq, int n_draft, int vocab) {
    return guarded<long long>([&] { return verify_ws(n_seq, n_draft, vocab); });
}

int mk_verify_drafts(int n_seq, int n_draft, int vocab, const void * target, long long row_stride, int dtype, int probs, const float * temperature,
                     const float * draft_probs, const int * drafts, const int * n_drafts, const float * u, int * accepted, int * tokens, float * draft_p,
                     void * ws, long long ws_bytes, void * stream) {
    return guarded<int>([&] {
        const unsigned sz = size_of(dtype);
        const long long want = verify_ws(n_seq, n_draft, vocab);
        if (probs != 0 && probs != 1) bad("probs: 0 logits, 1 probabilities");
        if (probs && dtype != DT_F32) bad("probabilities are fp32");
        if (probs && temperature) bad("a temperature applies to logits");
        if (row_stride < vocab) bad("row_stride is less than vocab");
        if (!n_seq) return 0; // (an empty tensor's pointers are null)
        need(target, "target");
        need(u, "u");
        need(accepted, "accepted");
        need(tokens, "tokens");
        if (n_draft) need(drafts, "drafts");
        aligned(target, sz, "target");
        for (const void * p : {(const void *) temperature, (const void *) draft_probs, (const void *) drafts, (const void *) n_drafts, (const void *) u,
                               (const void *) accepted, (const void *) tokens, (const void *) draft_p})
            aligned(p, 4, "an array of 4-byte values");
        if (!ws || ws_bytes < want) bad("the call needs " + std::to_string(want) + " bytes of workspace (mk_verify_ws)");
        aligned(ws, 16, "ws");
        const Device d(stream);
        d.holds(target, "target");
        d.holds(temperature, "temperature");
        d.holds(draft_probs, "draft_probs");
        d.holds(drafts, "drafts");
        d.holds(n_drafts, "n_drafts");
        d.holds(u, "u");
        d.holds(accepted, "accepted");
        d.holds(tokens, "tokens");
        d.holds(draft_p, "draft_p");
        d.holds(ws, "ws");
        VerifyArgs a{};
        a.target = target;
        a.temp = temperature;
        a.q = draft_probs;
        a.drafts = drafts;
        a.n_drafts = n_drafts;
        a.u = u;
        a.accepted = accepted;
        a.tokens = tokens;
        a.p = draft_p;
        a.row_stride = row_stride;
        a.n_seq = n_seq;
        a.n = n_draft;
        a.vocab = vocab;
        a.nsl = slices(vocab);
        a.part = static_cast<VerifyPart *>(ws);
        a.rest = reinterpret_cast<double *>(a.part + (size_t) n_seq * (n_draft + 1) * a.nsl);
        ck(launch_verify(a, dtype, probs != 0, static_cast<hipStream_t>(stream)), "verify");
        return 0;
    });
}

} // extern "C"
