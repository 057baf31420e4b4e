// mjt_head_norm_rope and its gradient (kernels/head_norm_rope.h).
#include "common.h"

namespace mjt {

namespace {
void* g_part = nullptr;               // the workgroups' partial sums of the scales' gradients (guarded by the library's lock, as the scratch memory)
size_t g_part_bytes = 0;
void forget() {
    if (g_part && !ctx().dry_run) (void)hipFree(g_part);
    g_part = nullptr;
    g_part_bytes = 0;
}
const bool g_registered = (at_shutdown(&forget), true);

struct Plan {
    int type, scale_type, V, LP, NC;
    int64_t tokens, heads, dim;
    std::string name, defines;
    std::vector<uint64_t> args;        // words 0 .. 17; the results' are the caller's
};

// Checks what both directions have in common and chooses vectors and lanes.  `parts`: q, k and v or their gradients (null: left out).
Plan plan_for(const char* who, const mjt_tensor* x, const mjt_tensor* q_scale, const mjt_tensor* k_scale, const mjt_tensor* table, const mjt_tensor* positions,
              const mjt_head_norm* p, const mjt_tensor* const parts[3], const mjt_tensor* dx, bool back) {
    require_init();
    MJT_CHECK(p, who << ": null parameters");
    check_tensor(x, who);
    Plan a;
    a.type = element_type(x->dtype);
    if (a.type < 0) MJT_FAIL(MJT_ERR_UNSUPPORTED, who << ": dtype " << mjt_dtype_name(x->dtype));
    MJT_CHECK(x->ndim >= 3, who << ": x has to be [.., tokens, heads, dim], got " << shape_str(x));
    const int64_t H = x->shape[x->ndim - 2], D = x->shape[x->ndim - 1], S = x->shape[x->ndim - 3];
    MJT_CHECK(p->q_heads >= 0 && p->k_heads >= 0 && p->v_heads >= 0 && (int64_t)p->q_heads + p->k_heads + p->v_heads == H,
              who << ": " << p->q_heads << " + " << p->k_heads << " + " << p->v_heads << " heads in " << shape_str(x));
    a.heads = H;
    a.dim = D;
    a.tokens = 1;
    for (int i = 0; i < x->ndim - 2; i++) a.tokens *= x->shape[i];
    MJT_CHECK(D >= 2 && D % 2 == 0, who << ": heads of " << D << " elements (an even number is needed)");
    MJT_CHECK(a.tokens < (int64_t(1) << 31) && H < (int64_t(1) << 24), who << ": too many tokens or heads in " << shape_str(x));
    const int64_t counts[3] = {p->q_heads, p->k_heads, p->v_heads};
    for (int i = 0; i < 3; i++)
        if (parts[i]) {
            check_tensor(parts[i], who);
            MJT_CHECK(parts[i]->dtype == x->dtype && numel(parts[i]) == a.tokens * counts[i] * D, who << ": part " << i << " is " << shape_str(parts[i]) << " or of another dtype");
        }
    if (dx) {
        check_tensor(dx, who);
        MJT_CHECK(dx->dtype == x->dtype && numel(dx) == numel(x), who << ": the gradient of x is " << shape_str(dx) << " or of another dtype");
    }
    // scales: both or neither (no norm)
    MJT_CHECK((q_scale == nullptr) == (k_scale == nullptr), who << ": scales for the queries and for the keys, or none");
    a.scale_type = a.type;
    if (q_scale) {
        for (const mjt_tensor* s : {q_scale, k_scale}) {
            check_tensor(s, who);
            MJT_CHECK(numel(s) == D && s->dtype == q_scale->dtype, who << ": a scale is " << shape_str(s) << ", heads have " << D << " elements; both have one dtype");
        }
        a.scale_type = element_type(q_scale->dtype);
        if (a.scale_type < 0) MJT_FAIL(MJT_ERR_UNSUPPORTED, who << ": scales of dtype " << mjt_dtype_name(q_scale->dtype));
    }
    MJT_CHECK(p->eps >= 0.0, who << ": eps " << p->eps);
    // the table and the positions
    int64_t rot = 0, rows = 0, per = 1;
    int axes = 1;
    std::string ends = "{0}";
    if (table) {
        check_tensor(table, who);
        MJT_CHECK(table->dtype == MJT_FLOAT32 && table->ndim == 3 && table->shape[2] == 2 && table->shape[1] >= 1 && table->shape[0] >= 1 && 2 * table->shape[1] <= D,
                  who << ": the table has to be float32 [positions, pairs, 2] with at most " << D / 2 << " pairs, got " << shape_str(table));
        rows = table->shape[0];
        rot = 2 * table->shape[1];
        MJT_CHECK(rows < (int64_t(1) << 31), who << ": a table of " << rows << " positions");
        MJT_CHECK(p->n_axes >= 0 && p->n_axes <= MJT_MOST_AXES, who << ": " << p->n_axes << " axes");
        if (p->n_axes) {
            axes = p->n_axes;
            int64_t sum = 0;
            ends = "{";
            for (int i = 0; i < axes; i++) {
                MJT_CHECK(p->sections[i] >= 0, who << ": a section of " << p->sections[i] << " pairs");
                sum += p->sections[i];
                ends += (i ? "," : "") + std::to_string(sum);
            }
            ends += "}";
            MJT_CHECK(sum == rot / 2, who << ": sections of " << sum << " pairs in all, the table has " << rot / 2);
            MJT_CHECK(positions, who << ": several axes need positions");
        } else
            ends = "{" + std::to_string(rot / 2) + "}";
    }
    if (positions) {
        check_tensor(positions, who);
        const int64_t n = numel(positions);
        MJT_CHECK(table && positions->dtype == MJT_INT32, who << ": positions are int32, with a table");
        // an axis has a position for every token, or for those of a sequence
        MJT_CHECK(n == axes * a.tokens || n == axes * S, who << ": " << n << " positions for " << axes << " axes of " << a.tokens << " tokens in sequences of " << S);
        per = n / axes;
    }
    // Vectors of 16 bytes where pairs, rows and pointers allow; of 16-bit elements 8 bytes in the backward pass and with several axes, where eight
    // pairs a lane take more registers than the wider access gives back (us for 8 / 4 pairs: 48 heads of 128, 8192 tokens, forward 41.4 / 44.8,
    // backward 64.2 / 63.3; 24 heads of 80 on three axes, 9477 tokens, 21.9 / 18.0 and 41.8 / 30.5).
    const int esz = dtype_size(x->dtype), ssz = q_scale ? dtype_size(q_scale->dtype) : 1;
    int V = back || axes > 1 ? 4 : 16 / esz;
    auto fits = [&](int v) {
        if ((rot / 2) % v || (D / 2) % v) return false;
        for (const mjt_tensor* t : {x, parts[0], parts[1], parts[2], dx})
            if (t && (uintptr_t)t->ptr % (size_t)(v * esz)) return false;
        return !q_scale || ((uintptr_t)q_scale->ptr % (size_t)(v * ssz) == 0 && (uintptr_t)k_scale->ptr % (size_t)(v * ssz) == 0);
    };
    while (V > 1 && !fits(V)) V /= 2;
    const int64_t chunks = D / 2 / V;
    int LP = 1;
    while (LP < chunks && LP < 64) LP *= 2;
    const int64_t NC = (chunks + LP - 1) / LP;
    if (NC * V > 32) MJT_FAIL(MJT_ERR_UNSUPPORTED, who << ": heads of " << D << " elements in vectors of " << V << " are not covered");
    a.V = V;
    a.LP = LP;
    a.NC = (int)NC;
    // Past the caches where every access of a wave takes whole lines of the rows, whose pieces lie as the kernel says (us through / past them: 8192 tokens of 48
    // heads of 128 bfloat16 42.2 / 38.3, gradient 63.6 / 59.6, on the other side 96 heads of 64 44.7 / 47.7 and 66.0 / 70.1, 48 of 128 with 64 elements turned 42.4 / 43.2, 9477
    // of 24 heads of 80 17.4 / 22.9); the gradient of heads turned in part also otherwise (48 of 128 with 64 turned 77.7 / 67.4).
    auto lines = [&](int64_t elements) { return elements * esz % 128 == 0; };
    const bool apart = V * esz >= 16, whole = p->interleaved ? lines(apart ? D / 2 : D) : lines(rot / 2) && lines(apart ? (D - rot) / 2 : D - rot);
    const bool far = (whole || (back && rot < D && lines(D))) && streams(a.tokens * H * D * esz * (back ? 3 : 2));
    std::ostringstream defs;
    defs << "#define STREAMS " << (far ? 1 : 0) << "\n#define TYPE " << a.type << "\n#define STYPE " << a.scale_type << "\n#define D " << D << "\n#define ROT " << rot << "\n#define V " << V << "\n#define LP " << LP << "\n#define NC " << NC
         << "\n#define PAIRED " << (p->interleaved ? 1 : 0) << "\n#define FIRST " << (p->heads_first ? 1 : 0) << "\n#define NORM " << (q_scale ? 1 : 0) << "\n#define AXES " << axes
         << "\n#define ENDS " << ends << "\n#define POS " << (positions ? 1 : 0) << "\n";
    a.defines = defs.str();
    a.name = std::string("mjt_head_norm_rope_") + mjt_dtype_name(x->dtype) + "_" + std::to_string(D) + (far ? "_streams" : "");
    auto ptr = [](const mjt_tensor* t) { return bits_of_ptr(t ? t->ptr : nullptr); };
    a.args = {ptr(x), ptr(parts[0]), ptr(parts[1]), ptr(parts[2]), ptr(q_scale), ptr(k_scale), ptr(table), ptr(positions), (uint64_t)a.tokens, (uint64_t)std::max<int64_t>(S, 1),
              (uint64_t)p->q_heads, (uint64_t)p->k_heads, (uint64_t)p->v_heads, bits_of(p->eps), (uint64_t)std::max<int64_t>(per, 1), (uint64_t)rows, 0, 0};
    return a;
}

void forward(const mjt_tensor* x, const mjt_tensor* q_scale, const mjt_tensor* k_scale, const mjt_tensor* table, const mjt_tensor* positions, const mjt_head_norm* p, const mjt_tensor* q,
             const mjt_tensor* k, const mjt_tensor* v) {
    const mjt_tensor* parts[3] = {q, k, v};
    Plan a = plan_for("head_norm_rope", x, q_scale, k_scale, table, positions, p, parts, nullptr, false);
    if (a.tokens == 0 || a.heads == 0) return;
    const int64_t rows = 64 / a.LP, rounds = (p->q_heads + rows - 1) / rows + (p->k_heads + rows - 1) / rows + (p->v_heads + rows - 1) / rows;
    // Few tokens: a wave for every round of every token.  Many: a wave for a token, three rounds under way together (us for 1 / 2 / 3 / 6 rounds: 48
    // heads of 128, 8192 tokens 47.1 / 43.3 / 41.4 / 45.3; 24 heads of 80, 9477 tokens 20.9 / 19.0 / 18.0 / 18.3).
    const bool few = a.tokens * rounds <= 4096;
    JitKernel* kern = layer_kernel(a.name, {"element.h", "head_norm_rope.h"}, a.defines + "#define BACK 0\n#define SUMS 0\n#define IT " + (few ? "1" : "3") + "\n");
    jit_launch(kern, (unsigned)std::min((a.tokens + 3) / 4, int64_t(1) << 20), few ? (unsigned)rounds : 1, 256, 0, a.args);
}

void backward(const mjt_tensor* x, const mjt_tensor* q_scale, const mjt_tensor* k_scale, const mjt_tensor* table, const mjt_tensor* positions, const mjt_head_norm* p, const mjt_tensor* dq,
              const mjt_tensor* dk, const mjt_tensor* dv, const mjt_tensor* dx, const mjt_tensor* dq_scale, const mjt_tensor* dk_scale) {
    const mjt_tensor* parts[3] = {dq, dk, dv};
    Plan a = plan_for("head_norm_rope_grad", x, q_scale, k_scale, table, positions, p, parts, dx, true);
    const bool sums = dq_scale || dk_scale;
    for (const mjt_tensor* s : {dq_scale, dk_scale})
        if (s) {
            check_tensor(s, "head_norm_rope_grad: a scale's gradient");
            MJT_CHECK(q_scale && numel(s) == a.dim && s->dtype == q_scale->dtype, "head_norm_rope_grad: a scale's gradient is " << shape_str(s) << " or of another dtype");
        }
    const bool nothing = a.tokens == 0 || a.heads == 0;
    if (nothing && !sums) return;
    const int64_t blocks = nothing ? 0 : std::min((a.tokens + 3) / 4, int64_t(1024));
    void* part = nullptr;
    if (sums) {
        const size_t bytes = (size_t)std::max<int64_t>(blocks, 1) * 2 * a.dim * 4;
        if (!ctx().dry_run && !grow_kept(&g_part, &g_part_bytes, bytes)) MJT_FAIL(MJT_ERR_DEVICE, "head_norm_rope_grad: no memory for partial sums");
        part = ctx().dry_run ? (void*)(uintptr_t)0x1000 : g_part;
    }
    if (!nothing) {
        a.args[16] = bits_of_ptr(dx ? dx->ptr : nullptr);
        a.args[17] = bits_of_ptr(part);
        JitKernel* kern = layer_kernel(a.name + "_grad", {"element.h", "head_norm_rope.h"}, a.defines + "#define BACK 1\n#define SUMS " + (sums ? "1" : "0") + "\n#define IT 3\n");
        jit_launch(kern, (unsigned)blocks, 1, 256, 0, a.args);
    }
    if (!sums) return;
    JitKernel* fold = layer_kernel("mjt_head_norm_rope_fold", {"element.h", "head_norm_rope.h"}, "#define FOLD 1\n#define STYPE " + std::to_string(a.scale_type) + "\n");
    jit_launch(fold, (unsigned)((2 * a.dim + 15) / 16), 1, 1024, 0,
               {bits_of_ptr(part), bits_of_ptr(dq_scale ? dq_scale->ptr : nullptr), bits_of_ptr(dk_scale ? dk_scale->ptr : nullptr), (uint64_t)blocks, (uint64_t)a.dim});
}
}  // namespace

}  // namespace mjt

extern "C" int mjt_head_norm_rope(const mjt_tensor* x, const mjt_tensor* q_scale, const mjt_tensor* k_scale, const mjt_tensor* table, const mjt_tensor* positions, const mjt_head_norm* p,
                                  const mjt_tensor* q, const mjt_tensor* k, const mjt_tensor* v) {
    return mjt::guarded([&] { mjt::forward(x, q_scale, k_scale, table, positions, p, q, k, v); });
}
extern "C" int mjt_head_norm_rope_grad(const mjt_tensor* x, const mjt_tensor* q_scale, const mjt_tensor* k_scale, const mjt_tensor* table, const mjt_tensor* positions, const mjt_head_norm* p,
                                       const mjt_tensor* dq, const mjt_tensor* dk, const mjt_tensor* dv, const mjt_tensor* dx, const mjt_tensor* dq_scale, const mjt_tensor* dk_scale) {
    return mjt::guarded([&] { mjt::backward(x, q_scale, k_scale, table, positions, p, dq, dk, dv, dx, dq_scale, dk_scale); });
}
