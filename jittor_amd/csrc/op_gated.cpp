// mjt_gated_linear and the element-wise part of its gradient; mjt_matmul_nearest.
#include "common.h"
#include <cmath>

namespace mjt {

void matmul_impl(const mjt_tensor* a, const mjt_tensor* b, const mjt_tensor* c, int trans_a, int trans_b, bool share_a);

namespace {
void* g_both = nullptr;               // gate and up of a call that does not want them (guarded by the library's lock, as the scratch memory)
size_t g_both_bytes = 0;
void forget() {
    if (g_both && !ctx().dry_run) (void)hipFree(g_both);
    g_both = nullptr;
    g_both_bytes = 0;
}
const bool g_registered = (at_shutdown(&forget), true);

const char* act_name(int act) {
    static const char* names[] = {"silu", "gelu", "relu", "sigmoid"};
    MJT_CHECK(act >= 0 && act < 4, "gated_linear: activation " << act);
    return names[act];
}

// gate and up [rows, 2 F] -> y [rows, F], or with dy [rows, F] -> d [rows, 2 F]
void rows_pass(int act, const void* both, const void* y, const void* d, int dtype, int64_t rows, int64_t F) {
    if (rows * F == 0) return;
    const size_t esz = (size_t)dtype_size(dtype);
    const bool wide = F % 4 == 0 && (uintptr_t)both % 16 == 0 && (uintptr_t)y % (4 * esz) == 0 && (uintptr_t)d % (4 * esz) == 0;
    const int V = wide ? 4 : 1;
    const std::string name = std::string("mjt_gated_") + act_name(act) + (d ? "_grad_" : "_") + mjt_dtype_name(dtype) + (wide ? "" : "_single");
    JitKernel* k = layer_kernel(name, {"element.h", "gated_act.h", "gated_rows.h"},
                                "#define TYPE " + std::to_string(element_type(dtype)) + "\n#define V " + std::to_string(V) + "\n#define ACT " + std::to_string(act) + "\n#define BACK " + (d ? "1" : "0") + "\n");
    const int64_t n = rows * F / V;
    jit_launch(k, (unsigned)std::min((n + 255) / 256, int64_t(1) << 23), 1, 256, 0, {bits_of_ptr(both), bits_of_ptr(y), bits_of_ptr(d), (uint64_t)n, (uint64_t)(F / V)});
}

bool forced(const char* route) {          // (a switch for measurements and tests: few, tiles or product)
    const char* e = getenv("MJT_GATED");
    return e && !strcmp(e, route);
}

// Up to 64 rows: one pass over the weights (kernels/gated_few.h).  False: not covered.
bool few_rows(const mjt_tensor* x, const mjt_tensor* w, int act, const mjt_tensor* y, const mjt_tensor* both) {
    const int64_t M = x->shape[0], K = x->shape[1], F = w->shape[0] / 2, esz = dtype_size(x->dtype);
    if (M > 64 || K == 0 || K * esz % 16 || K >= (int64_t(1) << 30) || F >= (int64_t(1) << 30) || (uintptr_t)x->ptr % 16 || (uintptr_t)w->ptr % 16 || (!forced("few") && getenv("MJT_GATED"))) return false;
    const int MB = (int)((M + 15) / 16), RB = 1, W = 4, UN = 4;
    std::ostringstream name, defs;
    name << "mjt_gated_few_" << act_name(act) << "_" << mjt_dtype_name(x->dtype) << "_" << MB * 16 << (both ? y ? "_both" : "_products" : "");
    defs << "#define TYPE " << element_type(x->dtype) << "\n#define ACT " << act << "\n#define W " << W << "\n#define RB " << RB << "\n#define MB " << MB << "\n#define UN " << UN << "\n#define BOTH "
         << (both ? 1 : 0) << "\n#define Y " << (y ? 1 : 0) << "\n";
    JitKernel* k = layer_kernel(name.str(), {"element.h", "gated_act.h", "gated_few.h"}, defs.str());
    jit_launch(k, (unsigned)((F + 16 * RB - 1) / (16 * RB)), 1, W * 64, 0,
               {bits_of_ptr(x->ptr), bits_of_ptr(w->ptr), bits_of_ptr(y ? y->ptr : nullptr), bits_of_ptr(both ? both->ptr : nullptr), (uint64_t)M, (uint64_t)F, (uint64_t)K});
    return true;
}

// 16-bit operands: gate and up on the same tiles of the matrix product's kernel (kernels/gemm_dma.h with GATED).  False: not covered.
bool on_tiles(const mjt_tensor* x, const mjt_tensor* w, int act, const mjt_tensor* y, const mjt_tensor* both) {
    Context& c = ctx();
    const int64_t M = x->shape[0], K = x->shape[1], F = w->shape[0] / 2;
    if (dtype_size(x->dtype) != 2 || K % 8 || K < 64 || K * 2 * 256 >= (int64_t(1) << 31) || M >= (int64_t(1) << 31) || F >= (int64_t(1) << 30) || (uintptr_t)x->ptr % 16 || (uintptr_t)w->ptr % 16 ||
        (!forced("tiles") && getenv("MJT_GATED")))
        return false;
    const int64_t cus = c.dry_run || c.prop.multiProcessorCount <= 0 ? 256 : c.prop.multiProcessorCount;
    int tile = 0;
    for (int t = 256; t >= 128 && !tile; t /= 2) {
        const int64_t tm = (M + t - 1) / t, tn = (F + t / 2 - 1) / (t / 2);
        const double edge = ((double)M * F) / ((double)tm * t * tn * (t / 2)), tiles = (double)tm * tn, util = tiles / (std::ceil(tiles / cus) * cus);
        if (t == 128 || (edge >= 0.85 && util >= 0.7 && K >= 256)) tile = t;
    }
    const int64_t tm = (M + tile - 1) / tile, tn = (F + tile / 2 - 1) / (tile / 2);
    const int nbuf = tile == 256 ? 2 : tm * tn > cus ? 2 : 4, wpe = tile == 128 && nbuf == 2 ? 2 : 1;
    auto whole = [&](int v) { return F % v == 0 && (!y || (uintptr_t)y->ptr % (size_t)(v * 2) == 0) && (!both || (uintptr_t)both->ptr % (size_t)(v * 4) == 0); };
    const int vs = whole(4) ? 4 : whole(2) ? 2 : 1, tail = K % 64 ? 1 : 0, gated = (y ? 1 : 0) + (both ? 2 : 0);
    std::ostringstream name, defs;
    name << "mjt_gated_tiles_" << act_name(act) << "_" << mjt_dtype_name(x->dtype) << "_" << tile << "x" << tile << (wpe == 2 ? "_direct2" : "_direct") << (tail ? "_tail" : "") << (both ? y ? "_both" : "_products" : "");
    defs << "#define VS " << vs << "\n#define IN " << element_type(x->dtype) << "\n#define OUT 2\n#define A_KCONT 1\n#define B_KCONT 1\n#define TILE " << tile << "\n#define NBUF " << nbuf << "\n#define WPE " << wpe
         << "\n#define GATED " << gated << "\n#define KTAIL " << tail << "\n#define ACT " << act << "\n";
    JitKernel* k = layer_kernel(name.str(), {"element.h", "gated_act.h", "gemm_dma.h"}, defs.str());
    // (as for the plain product: a build that moved registers aside behind the spelled-out reads is not run)
    if (k->spilled != 0 || k->agprs < 0 || k->agprs > tile * tile / 256) return false;
    jit_launch(k, (unsigned)((tm * tn + 7) / 8 * 8), 1, 256, 0,
               {bits_of_ptr(x->ptr), bits_of_ptr(w->ptr), bits_of_ptr(y ? y->ptr : nullptr), (uint64_t)M, (uint64_t)F, (uint64_t)K, (uint64_t)K, bits_of_ptr(both ? both->ptr : nullptr), 0, 0, 0, 0});
    return true;
}

void forward(const mjt_tensor* x, const mjt_tensor* w, int act, const mjt_tensor* y, const mjt_tensor* both) {
    require_init();
    act_name(act);
    check_tensor(x, "gated_linear: x");
    check_tensor(w, "gated_linear: the weights");
    MJT_CHECK(y || both, "gated_linear: no result is wanted");
    if (element_type(x->dtype) < 0) MJT_FAIL(MJT_ERR_UNSUPPORTED, "gated_linear: dtype " << mjt_dtype_name(x->dtype));
    MJT_CHECK(x->ndim == 2 && w->ndim == 2 && w->dtype == x->dtype && w->shape[1] == x->shape[1] && w->shape[0] % 2 == 0,
              "gated_linear: x " << shape_str(x) << " and weights " << shape_str(w) << " have to be [rows, k] and [2 f, k] of one dtype");
    const int64_t M = x->shape[0], F = w->shape[0] / 2;
    if (y) {
        check_tensor(y, "gated_linear: y");
        MJT_CHECK(y->ndim == 2 && y->dtype == x->dtype && y->shape[0] == M && y->shape[1] == F, "gated_linear: y is " << shape_str(y) << " or of another dtype");
    }
    if (both) {
        check_tensor(both, "gated_linear: gate and up");
        MJT_CHECK(both->ndim == 2 && both->dtype == MJT_FLOAT32 && both->shape[0] == M && both->shape[1] == 2 * F, "gated_linear: gate and up are " << shape_str(both) << " or not float32");
    }
    if (M == 0 || F == 0) return;
    if (few_rows(x, w, act, y, both) || on_tiles(x, w, act, y, both)) return;
    // the rest: both projections as one product in 32 bits, then the activation
    mjt_tensor c{};
    if (both) c = *both;
    else {
        const size_t bytes = (size_t)(M * 2 * F * 4);
        if (!ctx().dry_run && !grow_kept(&g_both, &g_both_bytes, bytes)) MJT_FAIL(MJT_ERR_DEVICE, "gated_linear: no memory for gate and up");
        c.ptr = ctx().dry_run ? (void*)(uintptr_t)0x1000 : g_both;
        c.dtype = MJT_FLOAT32;
        c.ndim = 2;
        c.shape[0] = M;
        c.shape[1] = 2 * F;
    }
    matmul_impl(x, w, &c, 0, 1, false);
    if (y) rows_pass(act, c.ptr, y->ptr, nullptr, y->dtype, M, F);
}

void backward(const mjt_tensor* dy, const mjt_tensor* both, int act, const mjt_tensor* d) {
    require_init();
    act_name(act);
    check_tensor(dy, "gated_linear_grad: dy");
    check_tensor(both, "gated_linear_grad: gate and up");
    check_tensor(d, "gated_linear_grad: d");
    if (element_type(dy->dtype) < 0) MJT_FAIL(MJT_ERR_UNSUPPORTED, "gated_linear_grad: dtype " << mjt_dtype_name(dy->dtype));
    MJT_CHECK(dy->ndim == 2 && both->ndim == 2 && d->ndim == 2 && both->dtype == MJT_FLOAT32 && d->dtype == dy->dtype && both->shape[0] == dy->shape[0] && d->shape[0] == dy->shape[0] &&
                  both->shape[1] == 2 * dy->shape[1] && d->shape[1] == both->shape[1],
              "gated_linear_grad: dy " << shape_str(dy) << ", gate and up " << shape_str(both) << ", d " << shape_str(d));
    rows_pass(act, both->ptr, dy->ptr, d->ptr, dy->dtype, dy->shape[0], dy->shape[1]);
}
}  // namespace

}  // namespace mjt

extern "C" int mjt_gated_linear(const mjt_tensor* x, const mjt_tensor* w, int activation, const mjt_tensor* y, const mjt_tensor* both) {
    return mjt::guarded([&] { mjt::forward(x, w, activation, y, both); });
}
extern "C" int mjt_gated_linear_grad(const mjt_tensor* dy, const mjt_tensor* both, int activation, const mjt_tensor* d) {
    return mjt::guarded([&] { mjt::backward(dy, both, activation, d); });
}
extern "C" int mjt_matmul_nearest(const mjt_tensor* a, const mjt_tensor* b, const mjt_tensor* c, int trans_a, int trans_b) {
    return mjt::guarded([&] {
        mjt::Nearest nearest;
        mjt::matmul_impl(a, b, c, trans_a, trans_b, false);
    });
}
