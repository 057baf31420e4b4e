// What the operators of transformer layers share (op_head_norm.cpp, op_gated.cpp, op_dropout.cpp): kernels by name and element types.
#include "common.h"
#include <mutex>
#include <unordered_map>

namespace mjt {

namespace {
std::mutex g_mu;
std::unordered_map<std::string, JitKernel*> g_kernels;
void forget() {   // the kernels belong to the run-time compiler's cache, which mjt_shutdown empties
    std::lock_guard<std::mutex> lock(g_mu);
    g_kernels.clear();
}
const bool g_registered = (at_shutdown(&forget), true);
}  // namespace

int element_type(int dtype) { return dtype == MJT_BFLOAT16 ? 0 : dtype == MJT_FLOAT16 ? 1 : dtype == MJT_FLOAT32 ? 2 : -1; }

JitKernel* layer_kernel(const std::string& name, std::initializer_list<const char*> files, const std::string& defines) {
    const std::string key = name + "|" + defines;
    {
        std::lock_guard<std::mutex> lock(g_mu);
        auto it = g_kernels.find(key);
        if (it != g_kernels.end()) return it->second;
    }
    std::string source = "#define ENTRY " + name + "\n" + defines;
    for (const char* f : files) source += std::string(embedded_source(f)) + "\n";
    JitKernel* k = jit_get(source, name);
    std::lock_guard<std::mutex> lock(g_mu);
    g_kernels.emplace(key, k);
    return k;
}

}  // namespace mjt
