// The experts' plan (step_moe_plan.h) on the host, for test_host_moe_plan.py.
#include PLAN

using namespace qkv;

static MoeArgs shape(int rows, int dim, int inner, int experts, int top, int gsh, int mins) {
    MoeArgs a{};
    a.rows = rows, a.dim = dim, a.inner = inner, a.n_experts = experts, a.top_k = top, a.gsh = gsh;
    a.up.mins = a.down.mins = mins ? reinterpret_cast<const uint16_t *>(8) : nullptr;
    return a;
}

extern "C" {
int model_holds(int rows, int dim, int inner, int experts, int top, int gsh, int mins, int xform) {
    MoeArgs a = shape(rows, dim, inner, experts, top, gsh, mins);
    split_work(a, xform);
    return plan_holds(a, xform);
}
int model_parts(int runs, int cr, int log) { return parts_hold(runs, cr, log); }
// every form of a number of rows and experts, the dims in turn from `at` on; the first shape that does not hold in `bad`; shapes looked at
long long model_sweep(int rows, int experts, int at, int * bad) {
    long long n = 0;
    for (int top = 1; top <= 16 && top <= experts; top++)
        for (int gsh = 0; gsh < 3; gsh++)
            for (int mins = 0; mins < 2; mins++)
                for (int xform : {(int) DT_F32, (int) DT_F16, (int) DT_BF16, (int) W4_UNITS})
                    for (int i = 0; i < 6; i++, n++) {
                        at = (int) ((at * 1103515245ll + 12345) & 0x7fffffff);
                        const int dim = 32 * (1 + (at >> 8) % (i < 3 ? 512 : 40)), inner = 32 * (1 + (at >> 12) % (i < 3 ? 1024 : 60));
                        if (model_holds(rows, dim, inner, experts, top, gsh, mins, xform)) continue;
                        const int b[] = {rows, dim, inner, experts, top, gsh, mins, xform};
                        for (int k = 0; k < 8; k++) bad[k] = b[k];
                        return -1;
                    }
    return n;
}
}
