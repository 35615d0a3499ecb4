// Checks of the arguments of the C ABI's operators around the recurrences (ops_api.hip, layer_api.hip).
#pragma once
#include "common.hpp"

namespace t2fw {

inline size_t size_of(int dtype) { return dtype == T2FW_F64 ? 8 : dtype == T2FW_F32 ? 4 : dtype == T2FW_F16 || dtype == T2FW_BF16 ? 2 : 0; }
inline size_t accumulator_size(int dtype) { return dtype == T2FW_F64 ? 8 : 4; }

inline int bad_dtype(int dtype) { return fail(T2FW_ERR_BAD_DTYPE, "unknown dtype code %d", dtype); }
inline int bad_workspace(size_t need, size_t given) { return fail(T2FW_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, given); }

struct Array {
    const char *name;
    const void *at;
    size_t align;
    bool optional;
};
inline int check_arrays(std::initializer_list<Array> arrays) {
    for (const Array &a : arrays) {
        if (a.at == nullptr) {
            if (a.optional) continue;
            return fail(T2FW_ERR_NULL_POINTER, "%s is a null pointer", a.name);
        }
        if (reinterpret_cast<uintptr_t>(a.at) % a.align != 0)
            return fail(T2FW_ERR_MISALIGNED, "%s is not aligned to %zu bytes", a.name, a.align);
    }
    return T2FW_OK;
}
// sizes whose product in bytes is addressable
inline int check_sizes(std::initializer_list<int64_t> sizes, const char *what) {
    long double bytes = 16;
    for (int64_t n : sizes) {
        if (n < 0) return fail(T2FW_ERR_BAD_SHAPE, "%s: sizes must be non-negative", what);
        bytes *= n > 0 ? (long double)n : 1;
    }
    if (bytes > 9.0e18L) return fail(T2FW_ERR_BAD_SHAPE, "%s: not addressable", what);
    return T2FW_OK;
}

}  // namespace t2fw
