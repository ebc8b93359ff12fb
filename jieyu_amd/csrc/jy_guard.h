// jy_guard.h — errors at the C ABI: thrown inside, turned into a status and the calling thread's
// jyhip_last_error() text at the entry point.
#pragma once

#include <hip/hip_runtime.h>

#include <exception>
#include <string>

namespace jy {

inline thread_local std::string g_err;

struct Error {
    std::string msg;
};

[[noreturn]] inline void fail(const std::string& m) { throw Error{m}; }

inline void ck(hipError_t e, const char* what) {
    if (e != hipSuccess) fail(std::string(what) + ": " + hipGetErrorString(e));
}

template <class F>
auto guarded(F&& f, decltype(f()) bad) -> decltype(f()) {
    try {
        g_err.clear();
        return f();
    } catch (const Error& e) {
        g_err = e.msg;
    } catch (const std::exception& e) {
        g_err = e.what();
    } catch (...) {
        g_err = "unknown error";
    }
    return bad;
}

}  // namespace jy

#define CK(x) ::jy::ck((x), #x)
