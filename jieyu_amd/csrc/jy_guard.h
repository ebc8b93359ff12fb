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

// `device` current for a call (the caller's is put back when it ends); a stream of another is refused
class OnDevice {
public:
    OnDevice(int device, hipStream_t st) {
        ck(hipGetDevice(&was_), "hipGetDevice");
        int on = device;
        if (st) ck(hipStreamGetDevice(st, &on), "hipStreamGetDevice");
        if (on != device) fail("the stream is on another device than the buffers");
        if (was_ != device) {
            ck(hipSetDevice(device), "hipSetDevice");
            set_ = true;
        }
    }
    ~OnDevice() {
        if (set_) (void)hipSetDevice(was_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;

private:
    int was_ = 0;
    bool set_ = false;
};

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
