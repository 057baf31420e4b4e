// mjt_dropout: dropout whose mask is worked out from the elements' places (kernels/dropout.h).
#include "common.h"
#include <cmath>

namespace mjt {

static void dropout_impl(const mjt_tensor* x, const mjt_tensor* residual, const mjt_tensor* y, double p, const mjt_fused_var* key, const mjt_fused_var* call, bool numbered) {
    require_init();
    check_tensor(x, "dropout: x");
    check_tensor(y, "dropout: y");
    const int type = element_type(x->dtype);
    if (type < 0) MJT_FAIL(MJT_ERR_UNSUPPORTED, "dropout: dtype " << mjt_dtype_name(x->dtype));
    const int64_t n = numel(x);
    MJT_CHECK(y->dtype == x->dtype && numel(y) == n, "dropout: x is " << shape_str(x) << ", y is " << shape_str(y) << " or of another dtype");
    if (residual) {
        check_tensor(residual, "dropout: residual");
        MJT_CHECK(residual->dtype == x->dtype && numel(residual) == n, "dropout: x is " << shape_str(x) << ", the residual is " << shape_str(residual) << " or of another dtype");
    }
    MJT_CHECK(p >= 0.0 && p <= 1.0, "dropout: a probability of " << p);
    MJT_CHECK(key && call && key->role == MJT_VAR_SCALAR && call->role == MJT_VAR_SCALAR, "dropout: the key and the call's number are scalars");
    if (n == 0) return;
    const uintptr_t group = 8 * (uintptr_t)dtype_size(x->dtype);
    const bool wide = (uintptr_t)x->ptr % group == 0 && (uintptr_t)y->ptr % group == 0 && (!residual || (uintptr_t)residual->ptr % group == 0);
    const bool far = streams(n * dtype_size(x->dtype) * (residual ? 3 : 2));
    const std::string name = "mjt_dropout_" + std::string(mjt_dtype_name(x->dtype)) + (numbered ? "" : "_unnumbered") + (residual ? "_residual" : "") + (wide ? "" : "_unaligned") + (far ? "_streams" : "");
    JitKernel* k = layer_kernel(name, {"element.h", "dropout.h"}, "#define TYPE " + std::to_string(type) + "\n#define RES " + (residual ? "1" : "0") + "\n#define WIDE " + (wide ? "1" : "0") + "\n#define SIDE " + (numbered ? "0u" : "0x10000000u") + "\n#define STREAMS " + (far ? "1" : "0") + "\n");
    const int64_t groups = (n + 7) / 8, blocks = std::min((groups + 255) / 256, int64_t(1) << 23);
    const uint64_t threshold = (uint64_t)std::nearbyint(p * 4294967296.0);
    jit_launch(k, (unsigned)blocks, 1, 256, 0, {bits_of_ptr(x->ptr), bits_of_ptr(residual ? residual->ptr : nullptr), bits_of_ptr(y->ptr), (uint64_t)n, (uint64_t)key->ivalue,
                                              (uint64_t)call->ivalue, threshold, bits_of(p < 1.0 ? 1.0 / (1.0 - p) : 0.0)});
}

}  // namespace mjt

extern "C" int mjt_dropout(const mjt_tensor* x, const mjt_tensor* residual, const mjt_tensor* y, double p, const mjt_fused_var* key, const mjt_fused_var* call) {
    return mjt::guarded([&] { mjt::dropout_impl(x, residual, y, p, key, call, true); });
}
extern "C" int mjt_dropout_unnumbered(const mjt_tensor* x, const mjt_tensor* residual, const mjt_tensor* y, double p, const mjt_fused_var* key, const mjt_fused_var* call) {
    return mjt::guarded([&] { mjt::dropout_impl(x, residual, y, p, key, call, false); });
}
