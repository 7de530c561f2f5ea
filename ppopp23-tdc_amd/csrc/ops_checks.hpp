// What the C entry points of the channels-last operators check alike.
#pragma once
#include <string>

#include "ops_internal.hpp"
#include "tdc_internal.hpp"

namespace tdc {

inline int invalid(const std::string &what) { return api_fail(TDC_ERR_INVALID, what); }
inline int launched(const char *what, int err) {
    return err ? api_fail(TDC_ERR_HIP, std::string(what) + ": " + hipGetErrorString((hipError_t)err)) : (int)TDC_OK;
}
inline bool number(int dtype) { return dtype == TDC_F32 || dtype == TDC_F16 || dtype == TDC_BF16; }
constexpr long long kMostItems = (1ll << 32) - 1;      // of a launch
inline bool aligned(const void *p, int bytes) { return ((uintptr_t)p & (unsigned)(bytes - 1)) == 0; }
inline int ws_check(const char *what, const void *ws, size_t have, size_t need) {
    if (!need) return TDC_OK;
    if (!ws || have < need)
        return invalid(std::string(what) + ": the workspace has " + std::to_string(ws ? have : 0) + " bytes, needs " + std::to_string(need));
    if (!aligned(ws, 16)) return invalid(std::string(what) + ": the workspace is not 16-byte aligned");
    return TDC_OK;
}
// (numbers in 4 or 8 bits)
inline int mx_range(const char *what, long long rows, long long K) {
    if (rows < 0 || K < 1) return invalid(std::string(what) + ": rows has to be 0 and K 1 at least");
    if (K > (1ll << 30) || rows > (1ll << 35) / mx4_padded(K) * 32) return invalid(std::string(what) + ": more numbers than 2^40");
    if (mx4_work_items(rows, K) > kMostItems) return invalid(std::string(what) + ": too many rows, a launch has fewer than 2^32 work items");
    return TDC_OK;
}
inline int mx_check(const char *what, long long rows, long long K, const void *codes, const void *scales) {
    if (int st = mx_range(what, rows, K)) return st;
    if (rows && (!codes || !scales)) return invalid(std::string(what) + ": null codes or scales");
    if (rows && (!aligned(codes, 16) || !aligned(scales, 16)))
        return invalid(std::string(what) + ": codes and scales have to be 16-byte aligned");
    return TDC_OK;
}

}  // namespace tdc

// (an error message is the only thing here that allocates: no exception leaves a C entry)
#define TDC_ENTRY try
#define TDC_ENTRY_END                 \
    catch (...) {                     \
        return (int)TDC_ERR_NOMEM;    \
    }
