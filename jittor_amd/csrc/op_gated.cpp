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
    const bool far = streams(rows * F * (8 + (d ? 3 : 1) * (int64_t)esz));
    const std::string name = std::string("mjt_gated_") + act_name(act) + (d ? "_grad_" : "_") + mjt_dtype_name(dtype) + (wide ? "" : "_single") + (far ? "_streams" : "");
    JitKernel* k = layer_kernel(name, {"element.h", "gated_act.h", "gated_rows.h"},
                                "#define TYPE " + std::to_string(element_type(dtype)) + "\n#define V " + std::to_string(V) + "\n#define ACT " + std::to_string(act) + "\n#define BACK " + (d ? "1" : "0") + "\n#define STREAMS " + (far ? "1" : "0") + "\n");
    const int64_t n = rows * F / V;
    jit_launch(k, (unsigned)std::min((n + 255) / 256, int64_t(1) << 23), 1, 256, 0, {bits_of_ptr(both), bits_of_ptr(y), bits_of_ptr(d), (uint64_t)n, (uint64_t)(F / V)});
}

// The ways to run the projections, by estimated time.
//   FEW (kernels/gated_few.h): up to 8 rows, and up to 16 where x is not the longer way: float32, whose MFMAs of other routes wait as well, and up to 48 MB of 16-bit weights
//   (us few / MFMA or TILES, weights not in the caches: bfloat16 8 x 4096 -> 11264 39.7 / 45.9, 8 x 2048 -> 5632 12.7 / 15.3, 16 x 2048 -> 5632 14.2 / 15.2, on the other side 16 x 4096 ->
//   11264 46.0 / 45.5, 16 x 2560 -> 6912 22.6 / 18.0; float32 16 x 4096 -> 4096 38.4 / 45.7; more sizes in profiles/gated_routes.txt).  Rows that are no whole 16-byte pieces, whose loads cross lines: 16 bits up to 20 MB,
//   float32 up to 8 rows or 48 MB (bfloat16 4 x 1501 -> 1500 9.7 / 12.3, 4 x 2231 -> 2610 22.3 / 16.7; float32 4 x 4001 -> 9001 84.8 / 98.3, 16 x 4001 -> 9001 114.7 / 99.8).
//   TILES (kernels/gemm_dma.h): 16-bit operands on 256 x 256 tiles, one to a compute unit, or 128 x 128, two to a unit.  Up to 128 rows only the latter (128 x 8192 -> 28672 235 /
//   188), up to 64 none: MFMA has tiles of 64 rows (us TILES / MFMA: 64 x 5120 -> 13824 62.9 / 57.5, 64 x 1536 -> 8960 20.1 / 18.9, 24 x 4096 -> 11264 42.2 / 42.1).
//   MFMA (kernels/gemm_mfma.h): any type and rows of any length; a product that is better cut into slices of its sum goes to PRODUCT, the plain product in
//   32 bits and a pass over it (before rows of any length ran here, us then / now: bfloat16 36 x 46 -> 256 23 / 5.7, 777 x 1001 -> 2600 42.1 / 32.8, 4000 x 45 -> 3001 67.7 / 30.7;
//   float32 3722 x 99 -> 3968 135 / 101, 1024 x 513 -> 1377 45.5 / 30.2).
// A stage of 64 elements of the sum takes 1.1 us on a 256 x 256 tile, 0.33 on a 128 x 128 tile with a unit to itself and 0.66 for two of them (more
// where the sum is long and neighbours drift apart), 0.25 on a 64 x 64 tile; a round begins with the first loads and ends with the
// activations and stores, 10, 6 and 3.5 us; a further round of tiles whose sum is long, a fifth more.  Left out: rows that are
// no whole 128-byte lines cost a quarter more on tiles, and weights that are not in the caches 5 us on tiles of 128 (80 to 128 rows would be MFMA's then).
// us measured 256 / 128 / MFMA for bfloat16, weights in the caches where they fit: 64 x 2048 -> 5632 43 / 16.3 / 11.3; 256 x 2048 -> 5632 45 / 17.5 / 22.4; 1024 x 2048 -> 5632 49.7 / 54.5 / 54.4; 2048 x
// 2048 -> 5632 103.6 / 92.4 / 106; 8192 x 2048 -> 5632 335 / 367 / 393; 512 x 4096 -> 11264 107 / 134 / 106; 777 x 1000 -> 2600 34.5 / 22.8 / 25.8; 512 x 1024 -> 2816
// 28.5 / 11.5 / 13.9; 4096 x 512 -> 1376 23.0 / 20.2 / 24.1.
enum Route { FEW, TILES, MFMA, PRODUCT };
Route choose(int dtype, int64_t M, int64_t F, int64_t K, bool aligned, int* tile) {
    const int64_t esz = dtype_size(dtype), cus = ctx().dry_run || ctx().prop.multiProcessorCount <= 0 ? 256 : ctx().prop.multiProcessorCount;
    const char* forced = getenv("MJT_GATED");                  // (a switch for measurements and tests; a route that does not cover the call is left out all the same)
    auto may = [&](const char* name) { return !forced || !strcmp(forced, name); };
    if (K == 0) return PRODUCT;
    const int64_t bytes = 2 * F * K * esz;
    const double stages = std::ceil((double)K / 64.0);
    auto rounds = [&](double tiles, double at_once) { return std::ceil(tiles / at_once); };
    auto tiles_of = [&](int64_t rows, int64_t cols) { return (double)((M + rows - 1) / rows) * (double)((F + cols - 1) / cols); };
    const int64_t mb = int64_t(1) << 20;
    const bool few = aligned ? M <= 8 || esz == 4 || bytes <= 48 * mb : esz == 2 ? bytes <= 20 * mb : M <= 8 || bytes <= 48 * mb;
    if (may("few") && M <= 16 && F < (int64_t(1) << 25) && (forced || few)) return FEW;
    if (may("tiles") && aligned && esz == 2 && K >= 64 && K * 2 * 256 < (int64_t(1) << 31)) {
        const double r256 = rounds(tiles_of(256, 128), (double)cus), n128 = tiles_of(128, 64), r128 = rounds(n128, 2.0 * (double)cus);
        const double t256 = r256 * (10.0 + 1.1 * stages) * (r256 > 1 ? 1.2 : 1.0);
        const double t128 = n128 <= (double)cus ? 5.3 + 0.335 * stages : r128 * (6.0 + 0.66 * stages * (1.0 + std::max(0.0, stages - 32.0) / 64.0)) * (r128 > 1 && stages >= 32.0 ? 1.2 : 1.0);
        const double mfma = 3.5 + 0.25 * stages * (1.0 + 0.8 * (rounds(tiles_of(64, 32), (double)cus) - 1.0));
        *tile = M > 128 && t256 < t128 ? 256 : 128;
        if (const char* e = getenv("MJT_GEMM_DMA")) *tile = atoi(e) == 128 ? 128 : 256;
        if (forced || (M > 64 && (*tile == 256 ? t256 : t128) < mfma)) return TILES;
    }
    return may("mfma") ? MFMA : PRODUCT;
}

void few_rows(const mjt_tensor* x, const mjt_tensor* w, int act, const mjt_tensor* y, const mjt_tensor* both) {
    const int64_t M = x->shape[0], K = x->shape[1], F = w->shape[0] / 2;
    // Lines of 128 bytes that a wave takes at a time: the most for which every wave has the same number of runs (us for 1 / 2 / 4, bfloat16, one row, weights not in
    // the caches: 4096 -> 11264 34.4 / 34.1 / 32.2, 4096 -> 14336 45.6 / 44.8 / 38.3, 5120 -> 13824 48.0 / 44.1 / 46.2, 2560 -> 6912 14.5 / 14.7 / 15.9 (15.4 another time), 1536 -> 8960 11.6 / 11.8 / 13.0).
    // Four waves instead of eight: 37.9 / 36.0 / 37.3 for the first of these, 8192 -> 1024 20.3 instead of 12.6.
    const int W = 8;
    const int64_t turn = W * 128 / dtype_size(x->dtype);
    const int UN = K % (4 * turn) == 0 ? 4 : K % (2 * turn) == 0 ? 2 : 1;
    const bool ragged = K * dtype_size(x->dtype) % 16 != 0 || (uintptr_t)x->ptr % 16 != 0 || (uintptr_t)w->ptr % 16 != 0;
    std::ostringstream name, defs;
    name << "mjt_gated_few_" << act_name(act) << "_" << mjt_dtype_name(x->dtype) << (ragged ? "_ragged" : "") << (both ? y ? "_both" : "_products" : "");
    defs << "#define RAGGED " << (ragged ? 1 : 0) << "\n#define TYPE " << element_type(x->dtype) << "\n#define ACT " << act << "\n#define W " << W << "\n#define UN " << UN << "\n#define BOTH " << (both ? 1 : 0) << "\n#define Y " << (y ? 1 : 0) << "\n";
    JitKernel* k = layer_kernel(name.str(), {"element.h", "gated_act.h", "gated_few.h"}, defs.str());
    jit_launch(k, (unsigned)((F + 7) / 8), 1, W * 64, 0,
               {bits_of_ptr(x->ptr), bits_of_ptr(w->ptr), bits_of_ptr(y ? y->ptr : nullptr), bits_of_ptr(both ? both->ptr : nullptr), (uint64_t)M, (uint64_t)F, (uint64_t)K});
}

// False: the compiler made no build of it that can be run.
bool on_tiles(const mjt_tensor* x, const mjt_tensor* w, int act, const mjt_tensor* y, const mjt_tensor* both, int tile) {
    const int64_t M = x->shape[0], K = x->shape[1], F = w->shape[0] / 2, cus = ctx().dry_run || ctx().prop.multiProcessorCount <= 0 ? 256 : ctx().prop.multiProcessorCount;
    const int64_t tm = (M + tile - 1) / tile, tn = (F + tile / 2 - 1) / (tile / 2);
    const int nbuf = tile == 256 ? 2 : tm * tn > cus ? 2 : 4, wpe = tile == 128 && nbuf == 2 ? 2 : 1;
    auto whole = [&](int v) { return F % v == 0 && (!y || (uintptr_t)y->ptr % (size_t)(v * 2) == 0) && (!both || (uintptr_t)both->ptr % (size_t)(v * 4) == 0); };
    const int vs = whole(4) ? 4 : whole(2) ? 2 : 1, tail = K % 64 ? 1 : 0, gated = (y ? 1 : 0) + (both ? 2 : 0);
    const bool far = both && streams(M * F * 10);               // (y alone is what the next product reads)
    std::ostringstream name, defs;
    name << "mjt_gated_tiles_" << act_name(act) << "_" << mjt_dtype_name(x->dtype) << "_" << tile << "x" << tile << (wpe == 2 ? "_direct2" : "_direct") << (tail ? "_tail" : "") << (both ? y ? "_both" : "_products" : "");
    defs << "#define VS " << vs << "\n#define IN " << element_type(x->dtype) << "\n#define OUT 2\n#define A_KCONT 1\n#define B_KCONT 1\n#define TILE " << tile << "\n#define NBUF " << nbuf << "\n#define WPE " << wpe
         << "\n#define GATED " << gated << "\n#define KTAIL " << tail << "\n#define ACT " << act << "\n#define STREAMS " << (far ? 1 : 0) << "\n";
    JitKernel* k = layer_kernel(name.str(), {"element.h", "gated_act.h", "gemm_dma.h"}, defs.str());
    // (as for the plain product: a build that moved registers aside behind the spelled-out reads is not run)
    if (k->spilled != 0 || k->agprs < 0 || k->agprs > tile * tile / 256) return false;
    MJT_CHECK(tm * tn < (int64_t(1) << 23), "gated_linear: launch too large");
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
    const int64_t K = x->shape[1];
    MJT_CHECK(M < (int64_t(1) << 31) && F < (int64_t(1) << 26) && K < (int64_t(1) << 30), "gated_linear: x " << shape_str(x) << " and weights " << shape_str(w) << " are too large");
    int tile = 0;
    const Route route = choose(x->dtype, M, F, K, K * dtype_size(x->dtype) % 16 == 0 && (uintptr_t)x->ptr % 16 == 0 && (uintptr_t)w->ptr % 16 == 0, &tile);
    if (route == FEW) {
        few_rows(x, w, act, y, both);
        return;
    }
    if (route == TILES && on_tiles(x, w, act, y, both, tile)) return;
    if (route != PRODUCT && gemm_gated(x->dtype, act, act_name(act), x->ptr, w->ptr, y ? y->ptr : nullptr, both ? both->ptr : nullptr, M, F, K)) return;
    // the rest: both projections as one product in 32 bits, then the activation; where nobody wants the products, some rows at a time, so that
    // they take 256 MB at most (or a row)
    const int64_t most = both ? M : std::max(int64_t(1), (int64_t(256) << 20) / (2 * F * 4));
    const int64_t rows = std::min(M, most);
    void* mem = nullptr;
    if (!both) {
        if (!ctx().dry_run && !grow_kept(&g_both, &g_both_bytes, (size_t)(rows * 2 * F * 4))) MJT_FAIL(MJT_ERR_DEVICE, "gated_linear: no memory for gate and up");
        mem = ctx().dry_run ? (void*)(uintptr_t)0x1000 : g_both;
    }
    for (int64_t r = 0; r < M; r += rows) {
        mjt_tensor a = *x, c{};
        a.shape[0] = std::min(rows, M - r);
        a.ptr = (char*)x->ptr + r * K * dtype_size(x->dtype);
        c.ptr = both ? both->ptr : mem;
        c.dtype = MJT_FLOAT32;
        c.ndim = 2;
        c.shape[0] = a.shape[0];
        c.shape[1] = 2 * F;
        {
            Nearest nearest;                                   // (which takes rows of any length as they lie)
            matmul_impl(&a, w, &c, 0, 1, false);
        }
        if (y) rows_pass(act, c.ptr, (char*)y->ptr + r * F * dtype_size(y->dtype), nullptr, y->dtype, a.shape[0], F);
    }
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
